// The argument checks and launch plans of the operators over a key/value cache (csrc/host/dispatch_cache.cpp) without a device: launches write
// down what they were asked for, workspaces are addresses that nobody touches.  Built and driven by test_cache_cpu.py.
#include <cstdarg>
#include <cstdio>
#include <cstring>

#include "dispatch_cache.cpp"

namespace {
char g_message[1024];
const char *g_launch = "";
size_t g_workspace = 0;
bool g_no_workspace = false;
tracea_amd::QkNormArgs g_qk;
tracea_amd::CacheAppendArgs g_append;
tracea_amd::AttentionCachedArgs g_attention;
}  // namespace

extern "C" {
hipError_t hipGetDevice(int *d) { *d = 0; return hipSuccess; }
hipError_t hipSetDevice(int) { return hipSuccess; }
const char *hipGetErrorString(hipError_t) { return "?"; }
}

namespace tracea_amd {
std::mutex g_launches;
TraceaStatus fail(TraceaStatus st, const char *fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(g_message, sizeof(g_message), fmt, ap);
  va_end(ap);
  return st;
}
bool runtime_ready() { return true; }
int runtime_device_count() { return 2; }
const DeviceLimits &device_limits() { static DeviceLimits l; return l; }
void *train_scratch(int, hipStream_t, size_t bytes) { g_workspace = bytes; return g_no_workspace ? nullptr : (void *)0x7000000000ull; }
int launch_qk_norm_forward(const QkNormArgs &a, int, hipStream_t) { g_launch = "qk_norm"; g_qk = a; return 0; }
int launch_qk_norm_backward(const QkNormArgs &a, int, hipStream_t) { g_launch = "qk_norm_backward"; g_qk = a; return 0; }
int launch_cache_append(const CacheAppendArgs &a, int, hipStream_t) { g_launch = "append"; g_append = a; return 0; }
int launch_attention_cached(const AttentionCachedArgs &a, int, bool, hipStream_t) { g_launch = "attention"; g_attention = a; return 0; }
}  // namespace tracea_amd

using namespace tracea_amd;
extern "C" {
const char *stub_message() { return g_message; }
const char *stub_launch() { return g_launch; }
void stub_reset(int no_workspace) { g_launch = ""; g_message[0] = 0; g_workspace = 0; g_no_workspace = no_workspace != 0; }
long long stub_value(const char *what) {
  auto is = [&](const char *x) { return strcmp(what, x) == 0; };
  if (is("workspace")) return (long long)g_workspace;
  if (is("qk.vec")) return g_qk.vec;
  if (is("qk.lanes")) return g_qk.lanes;
  if (is("qk.beside")) return g_qk.beside;
  if (is("qk.blocks")) return g_qk.blocks;
  if (is("append.vec")) return g_append.vec;
  if (is("append.held")) return g_append.held;
  if (is("append.pages")) return g_append.pages;
  if (is("append.groups")) return g_append.groups;
  if (is("append.heads")) return g_append.heads;
  if (is("append.queries")) return g_append.queries;
  if (is("append.tokens_at_once")) return append_tokens_at_once(g_append.P);
  if (is("append.queries_at_once")) return kAppendQueries;
  if (is("rows")) return g_attention.rows;
  if (is("row_blocks")) return g_attention.row_blocks;
  if (is("workgroups")) return g_attention.workgroups;
  if (is("splits")) return g_attention.splits;
  if (is("shares")) return g_attention.shares;
  if (is("apart")) return g_attention.apart;
  if (is("line")) return g_attention.line;
  if (is("step")) return g_attention.step;
  if (is("slots")) return g_attention.slots;
  if (is("meta")) return (long long)(intptr_t)g_attention.meta;
  if (is("part_o")) return (long long)(intptr_t)g_attention.part_o;
  if (is("part_ml")) return (long long)(intptr_t)g_attention.part_ml;
  if (is("page_magic")) return g_attention.page_magic;
  if (is("M")) return g_attention.table.M;
  return -1;
}
// page_of, as the kernels ask it
int stub_page_of(const int *table, long long sb, int M, int N, int P, int b, long long slot) { return page_of(PageTable{table, sb, M, N, P}, b, slot); }

TraceaStatus tracea_qk_norm_rotary(TraceaTensorView q, const TraceaTensorView *k, const TraceaTensorView *qw, const TraceaTensorView *kw,
                                   const TraceaTensorView *p, const TraceaTensorView *f, TraceaTensorView *qo, TraceaTensorView *ko, TraceaQkNormParams params) {
  return dispatch_qk_norm(q, k, qw, kw, p, f, qo, ko, params);
}
TraceaStatus tracea_qk_norm_rotary_backward(TraceaTensorView dqo, const TraceaTensorView *dko, TraceaTensorView q, const TraceaTensorView *k,
                                            const TraceaTensorView *qw, const TraceaTensorView *kw, const TraceaTensorView *p, const TraceaTensorView *f,
                                            TraceaTensorView *dq, TraceaTensorView *dk, TraceaTensorView *dqw, TraceaTensorView *dkw, TraceaQkNormParams params) {
  return dispatch_qk_norm_backward(dqo, dko, q, k, qw, kw, p, f, dq, dk, dqw, dkw, params);
}
TraceaStatus tracea_cache_append(TraceaTensorView k, TraceaTensorView v, const TraceaTensorView *q, TraceaTensorView *kc, TraceaTensorView *vc,
                                 TraceaTensorView *ks, TraceaTensorView *vs, TraceaTensorView pt, TraceaTensorView st, const TraceaTensorView *ln,
                                 const TraceaTensorView *p, const TraceaTensorView *f, TraceaTensorView *qo, TraceaCacheAppendParams params) {
  return dispatch_cache_append(k, v, q, kc, vc, ks, vs, pt, st, ln, p, f, qo, params);
}
TraceaStatus tracea_attention_cached(TraceaTensorView q, TraceaTensorView kc, TraceaTensorView vc, const TraceaTensorView *ks, const TraceaTensorView *vs,
                                     TraceaTensorView pt, const TraceaTensorView *ql, TraceaTensorView kl, TraceaTensorView *o, TraceaTensorView *lse,
                                     TraceaAttentionParams params) {
  return dispatch_attention_cached(q, kc, vc, ks, vs, pt, ql, kl, o, lse, params);
}
}
