// Argument checks and launches of the operators for training: attention with row statistics and its backward pass, rotary
// positions, the norm / gate / residual sum.  Status codes as in dispatch.cpp.
#include <cmath>

#include "operands.hpp"

namespace tracea_amd {

std::mutex g_launches;

namespace {

// ---- attention ------------------------------------------------------------------------------------------------

constexpr long long kMostBlocks = 1ll << 24;  // workgroups of 256 threads in a launch: fewer than 2^32 threads

struct Attention {
  const char *op;
  View q, k, v, o, lse, d_o, dq, dk, dv;
  View q_lengths, k_lengths;  // without elements where absent
  const int *q_len = nullptr, *k_len = nullptr;
  bool backward = false;
  float scale = 0.0f;
  int causal = 0;
  hipStream_t stream = nullptr;
};

TraceaStatus read_lengths(const char *op, const char *name, const TraceaTensorView *t, long long B, int device, View &v, const int **out) {
  if (t == nullptr) return TRACEA_SUCCESS;
  TraceaStatus st = read(op, name, *t, 1, &v);
  if (st != TRACEA_SUCCESS) return st;
  if (v.dtype != TRACEA_DTYPE_INT32 || v.shape[0] != B || (B > 1 && v.stride[0] != 1))
    return fail(TRACEA_INVALID_PARAMS, "%s: %s must be a contiguous i32 tensor of %lld entries, one per batch entry", op, name, B);
  if (v.device != device) return fail(TRACEA_INVALID_PARAMS, "%s: operands live on different devices", op);
  *out = (const int *)v.ptr;
  return TRACEA_SUCCESS;
}

// What the kernels read and write where it lies.
bool rows_in_place(const View &t, long long D) {
  return D % 8 == 0 && (t.stride[3] == 1 || t.shape[3] == 1) && t.stride[0] % 8 == 0 && t.stride[1] % 8 == 0 && t.stride[2] % 8 == 0 &&
         t.stride[1] >= 0 && t.stride[2] >= 0 && aligned(t.ptr, 16);
}

// Rows of a workgroup and parts of the keys for the forward pass, by the least of this estimate (us) over the candidates, in the terms of
// plan_backward and of how fast the keys can arrive: few rows over many keys leave CUs idle unless the keys are shared, by two waves of a
// workgroup (blocks of 64 rows, of 32 for at most 16 rows) or by workgroups, whose results a second launch joins.  Fitted to 34 shapes with every
// candidate timed; its choice is 2 % behind the best on average and 16 % at worst (of 6 us).  Best / unsplit blocks of 128, us: B1 H12 S1024
// D64 causal 15.4 / 21.9 (blocks of 64), B8 H32:8 one query over up to 8192 keys 46 / 167 (8 parts of blocks of 128; 4 of 32: 52; keys
// from HBM), B1 H40:8 one query over 32768 keys 34 / 642 (24 parts of blocks of 32), B1 H8 1000 queries over 5000 keys D64 30 / 63 (4 parts).
struct ForwardPlan {
  int block, splits;
};
ForwardPlan plan_forward(long long heads, long long rows, long long keys, int width, bool half, bool lengths, int cus) {
  ForwardPlan best{128, 1};
  double least = 1e300;
  const double f = width / 128.0, tiles = (double)((keys + 63) / 64), seen = half ? 0.5 : 1.0;
  for (int block : {128, rows > 16 ? 64 : 32})
    for (int splits : {1, 2, 3, 4, 6, 8, 12, 16, 24, 32}) {
      const int step = block < 128 ? 2 : 1;  // tiles
      const double bytes = 2.0 * splits * heads * rows * width * 4;
      if (tiles < step || (splits > 1 && (tiles < step * splits || bytes > (1 << 30)))) continue;
      const double lat = (block == 128 ? 1.37 : block == 64 ? 0.88 : 0.72) * (0.14 + 0.86 * f);
      const double thr = (block == 128 ? 0.81 : block == 64 ? 0.94 : 0.68) * f / cus, fill = rows < block ? 0.22 + 0.78 * rows / block : 1.0;
      const double n = (double)((rows + block - 1) / block) * heads * splits, walk = tiles / splits;
      const double slots = cus * (block == 128 || width == 64 ? 2.0 : 1.0);
      const double arrive = 4.0 * heads * keys * width * seen / 6e6 * std::max(1.0, 0.34 * slots / n) *
                            (lengths && block == 32 && width > 64 ? 1.2 : 1.0);  // (one workgroup on a CU: idle where its sequence has ended)
      const double total = thr * fill * n * (walk * seen + 2.2), longest = std::max(lat * (walk + 2.2), arrive);
      const double time = std::max(total, longest) + 0.42 * std::min(total, longest) + (splits > 1 ? 3.5 + bytes / 5.3e6 : 0.0);
      if (time < least) {
        least = time;
        best = {block, splits};
      }
    }
  return best;
}

// Columns of a workgroup and parts of the rows for dK and dV, by the least of this estimate (us) over the candidates.  A tile of 64 costs a
// workgroup of four waves `lat` while it walks and a CU `thr` of its throughput; blocks of 64 columns, two waves on 32, do half the
// work of blocks of 128 in 0.72 of the time.  The device is busy for the sum of all walks, but no shorter than the longest.  Parts are written and read as
// fp32 and summed in a launch of their own.  Fitted to 22 shapes with every candidate timed; its choice is 0.6 % behind the
// best on average and 6 % at worst.  Best / unsplit blocks of 128, us: B1 H12 S1024 D64 causal 26.5 / 37 (blocks of 64), B1 H8:1 S4096 D128
// causal 149 / 1500 (16 parts), B2 H32:8 S2048 D128 causal 243 / 380 (2 parts), B1 H16:2 S1024 D128 55 / 360 (16 parts).
struct BackwardPlan {
  int block, row_splits;
};
BackwardPlan plan_backward(long long heads, long long rows, long long keys, int width, bool causal, int cus) {
  BackwardPlan best{128, 1};
  double least = 1e300;
  const double f = width / 128.0, row_tiles = (double)((rows + 63) / 64), key_tiles = (double)((keys + 63) / 64), seen = causal ? 0.5 : 1.0;
  for (int block : {128, 64})
    for (int parts : {1, 2, 3, 4, 6, 8, 12, 16}) {
      const double bytes = (2.0 * parts + 1) * heads * keys * 2 * width * 4;
      if (parts > 1 && (row_tiles < 2 * parts || bytes > (1 << 30))) continue;
      const double lat = (block == 128 ? 2.5 : 1.8) * (0.05 + 0.95 * f), thr = (block == 128 ? 1.6 : 1.13) * (0.23 + 0.77 * f) / cus;
      const double n_k = (double)((keys + block - 1) / block) * heads * parts, n_q = (double)((rows + block - 1) / block) * heads;
      const double walk = row_tiles / parts;
      const double total = thr * (n_k * (walk * seen + 1.5) + n_q * (key_tiles * seen + 1.5) * 0.56);
      const double longest = lat * std::max(walk + 1.5, (key_tiles + 1.5) * 0.5);
      const double time = std::max(total, longest) + 0.27 * std::min(total, longest) + (parts > 1 ? 4.6 + bytes / 5.6e6 : 0.0);
      if (time < least) {
        least = time;
        best = {block, parts};
      }
    }
  return best;
}

TraceaStatus too_many(const char *op) { return fail(TRACEA_UNSUPPORTED_CONFIG, "%s: more workgroups than a launch can have", op); }

TraceaStatus run_attention(const Attention &c, bool from_copies) {
  const long long B = c.q.shape[0], Hq = c.q.shape[1], Sq = c.q.shape[2], D = c.q.shape[3], Hk = c.k.shape[1], Sk = c.k.shape[2];
  const long long G = Hq / Hk, rows_pad = (G * Sq + 63) / 64 * 64;
  DeviceScope scope(c.q.device);
  if (scope.err != hipSuccess) return hip_status("hipSetDevice", (int)scope.err);

  const View *reads[5] = {&c.q, &c.k, &c.v, &c.o, &c.d_o};
  const View *writes[3] = {&c.o, nullptr, nullptr};
  const int n_reads = c.backward ? 5 : 3;
  int n_writes = 1;
  if (c.backward) {
    writes[0] = &c.dq; writes[1] = &c.dk; writes[2] = &c.dv;
    n_writes = 3;
  }
  // (offsets inside a streamed tile are 32-bit: 64 keys, or 64 packed rows of a group's heads)
  auto tile_fits = [](long long rows, const View &t, long long heads) {
    return (rows * t.stride[2] + heads * t.stride[1] + 128) * 2 < (1ll << 31);
  };
  bool in_place = tile_fits(64, c.k, 0) && tile_fits(64, c.v, 0);
  if (c.backward) in_place = in_place && tile_fits(64 / G + 2, c.q, G) && tile_fits(64 / G + 2, c.d_o, G);
  for (int i = 0; i < n_reads; ++i) in_place = in_place && rows_in_place(*reads[i], D);
  for (int i = 0; i < n_writes; ++i) {
    in_place = in_place && rows_in_place(*writes[i], D);
    for (int j = 0; j < n_reads; ++j) in_place = in_place && !may_overlap(*writes[i], *reads[j]);
  }
  if (!in_place) {
    const long long Dp = (D + 7) / 8 * 8;
    const size_t one_q = (size_t)(B * Hq * Sq) * (size_t)Dp * 2, one_k = (size_t)(B * Hk * Sk) * (size_t)Dp * 2;
    const size_t bytes = c.backward ? 4 * one_q + 4 * one_k : 2 * one_q + 2 * one_k;
    unsigned char *buf = from_copies ? nullptr : (unsigned char *)train_copies(c.q.device, c.stream, bytes);
    if (buf == nullptr)
      return fail(TRACEA_UNSUPPORTED_CONFIG,
                  "%s: head dim %lld / these strides need padded copies, and no buffer for them can be had (stream under capture, "
                  "or above 1 GiB); in place: head dim a multiple of 8, contiguous, other strides multiples of 8 elements, bases "
                  "16-byte aligned, results over no operand", c.op, D);
    Attention p = c;
    auto dense = [&](View *t, size_t bytes_of) {
      t->ptr = buf;
      buf += bytes_of;
      t->shape[3] = Dp;
      t->stride[3] = 1;
      t->stride[2] = Dp;
      t->stride[1] = t->shape[2] * Dp;
      t->stride[0] = t->shape[1] * t->stride[1];
    };
    dense(&p.q, one_q); dense(&p.k, one_k); dense(&p.v, one_k); dense(&p.o, one_q);
    View *copies[5] = {&p.q, &p.k, &p.v, &p.o, &p.d_o};
    if (c.backward) {
      dense(&p.d_o, one_q); dense(&p.dq, one_q); dense(&p.dk, one_k); dense(&p.dv, one_k);
    }
    for (int i = 0; i < n_reads; ++i) {
      const View &s = *reads[i];
      if (count_of(s) == 0) continue;
      const long long rows = s.shape[0] * s.shape[1] * s.shape[2];
      const int e = launch_pad_copy(s.ptr, copies[i]->ptr, 2, rows, D, s.stride[0], s.stride[3], rows, Dp, c.stream, s.shape[1],
                                    s.stride[1], s.shape[2], s.stride[2]);
      if (e != 0) return hip_status("operand copy launch", e);
    }
    const TraceaStatus st = run_attention(p, true);
    if (st != TRACEA_SUCCESS) return st;
    const View *results[3] = {c.backward ? &p.dq : &p.o, &p.dk, &p.dv};
    for (int i = 0; i < n_writes; ++i) {
      const View &t = *writes[i];
      if (count_of(t) == 0) continue;
      const int e = launch_unpad_copy(results[i]->ptr, t.ptr, 2, t.shape[0] * t.shape[1] * t.shape[2], D, t.stride[0], t.stride[3], Dp,
                                      c.stream, t.shape[1], t.stride[1], t.shape[2], t.stride[2]);
      if (e != 0) return hip_status("result copy launch", e);
    }
    return TRACEA_SUCCESS;
  }

  AttentionTrainArgs a{};
  a.q = head_view(c.q); a.k = head_view(c.k); a.v = head_view(c.v); a.o = head_view(c.o);
  a.lse = (float *)c.lse.ptr;
  a.lse_sb = c.lse.stride[0]; a.lse_sh = c.lse.stride[1]; a.lse_ss = c.lse.stride[2];
  a.q_len = c.q_len; a.k_len = c.k_len;
  a.B = (int)B; a.Hk = (int)Hk; a.G = (int)G; a.Sq = (int)Sq; a.Sk = (int)Sk; a.D = (int)D;
  a.g_magic = G > 1 ? (unsigned)(((1ull << 32) + G - 1) / G) : 0;
  a.negate = c.scale < 0.0f;
  a.scale = fabsf(c.scale);
  a.scale_log2 = a.scale * 1.4426950408889634f;
  a.causal = c.causal;
  a.rows_pad = (int)rows_pad;
  a.order = c.q_len != nullptr || c.k_len != nullptr ? 2 : c.causal ? 1 : 0;
  a.splits = 1;
  if (!c.backward) {
    if (Sq == 0) return TRACEA_SUCCESS;
    const int width = D <= 64 ? 64 : D <= 96 ? 96 : 128;
    const ForwardPlan plan = plan_forward(B * Hk, G * Sq, Sk, width, a.causal && Sq == Sk, c.k_len != nullptr, (int)device_limits().cus);
    a.block = plan.block;
    if (B * Hk * ((G * Sq + a.block - 1) / a.block) >= kMostBlocks) return too_many(c.op);
    if (plan.splits > 1) {
      const long long keys = a.block < 128 ? 128 : 64, steps = (Sk + keys - 1) / keys, per = (steps + plan.splits - 1) / plan.splits;
      const long long splits = (steps + per - 1) / per;
      const size_t n = (size_t)(splits * B * Hk * G * Sq);
      a.part_o = (float *)train_scratch(c.q.device, c.stream, n * (size_t)(width + 2) * 4);
      if (a.part_o != nullptr) {  // (else unsplit: slower, the same result to rounding)
        a.part_ml = a.part_o + n * width;
        a.splits = (int)splits;
        a.steps_per_split = (int)per;
      }
    }
    return hip_status("attention forward launch", launch_attention_train_forward(a, c.q.dtype, c.stream));
  }
  a.d_o = head_view(c.d_o); a.dq = head_view(c.dq); a.dk = head_view(c.dk); a.dv = head_view(c.dv);
  const size_t stats = (size_t)(B * Hk * rows_pad);
  a.norm_blocks = c.q.dtype == TRACEA_DTYPE_FLOAT16 ? (int)(rows_pad / 64 + (Sk + 63) / 64) : 0;
  const size_t width = D <= 64 ? 64 : D <= 96 ? 96 : 128;
  const size_t norms = ((size_t)(B * Hk) * a.norm_blocks + 3) / 4 * 4;
  const BackwardPlan plan = plan_backward(B * Hk, G * Sq, Sk, (int)width, a.causal, (int)device_limits().cus);
  a.block = plan.block;
  a.row_splits = plan.row_splits;
  auto blocks = [&](long long n, long long of) { return B * Hk * ((n + of - 1) / of); };
  if (blocks(Sk, a.block) * a.row_splits + blocks(G * Sq, a.block) >= kMostBlocks || blocks(rows_pad + Sk + 63, 64) >= kMostBlocks ||
      (a.row_splits > 1 && blocks(Sk * 2 * (long long)width / 4, 1) / 256 >= kMostBlocks))
    return too_many(c.op);
  auto workspace = [&]() {
    const size_t parts = a.row_splits > 1 ? (size_t)a.row_splits * (size_t)(B * Hk * Sk) * 2 * width : 0;
    return (float *)train_scratch(c.q.device, c.stream, (2 * stats + norms + parts + 1) * 4);
  };
  float *ws = workspace();
  if (ws == nullptr && a.row_splits > 1) {  // (slower without the parts, the same sums to rounding)
    a.row_splits = 1;
    ws = workspace();
  }
  if (ws == nullptr)
    return fail(TRACEA_UNSUPPORTED_CONFIG, "%s: no workspace can be had (a stream under capture that made no such call before, or out of "
                                           "memory)", c.op);
  a.neg_lse2 = ws;
  a.neg_delta = ws + stats;
  a.norms = ws + 2 * stats;
  a.part_dkv = a.norms + norms;
  return hip_status("attention backward launch", launch_attention_train_backward(a, c.q.dtype, c.stream));
}

TraceaStatus check_attention(Attention &c, const TraceaAttentionParams &params, const TraceaTensorView *q_lengths,
                             const TraceaTensorView *k_lengths, bool *nothing) {
  const char *op = c.op;
  *nothing = false;
  if (!is_half(c.q.dtype)) return fail(TRACEA_UNSUPPORTED_CONFIG, "%s: f16 or bf16 tensors (got %s)", op, dtype_name(c.q.dtype));
  const View *halves[7] = {&c.k, &c.v, &c.o, &c.d_o, &c.dq, &c.dk, &c.dv};
  for (int i = 0; i < (c.backward ? 7 : 3); ++i)
    if (halves[i]->dtype != c.q.dtype) return fail(TRACEA_UNSUPPORTED_CONFIG, "%s: all tensors but lse must share one type, f16 or bf16", op);
  if (c.lse.dtype != TRACEA_DTYPE_FLOAT32) return fail(TRACEA_INVALID_PARAMS, "%s: lse must be f32", op);
  const long long B = c.q.shape[0], Hq = c.q.shape[1], Sq = c.q.shape[2], D = c.q.shape[3], Hk = c.k.shape[1], Sk = c.k.shape[2];
  if (c.k.shape[0] != B || c.k.shape[3] != D || !same_shape(c.k, c.v) || !same_shape(c.q, c.o) ||
      (c.backward && (!same_shape(c.q, c.d_o) || !same_shape(c.q, c.dq) || !same_shape(c.k, c.dk) || !same_shape(c.k, c.dv))))
    return fail(TRACEA_INVALID_PARAMS, "%s: q, o (d_o, dq) must be [B,Hq,Sq,D], k, v (dk, dv) [B,Hk,Sk,D]", op);
  if (c.lse.shape[0] != B || c.lse.shape[1] != Hq || c.lse.shape[2] != Sq)
    return fail(TRACEA_INVALID_PARAMS, "%s: lse must be [B,Hq,Sq]", op);
  TraceaStatus st = check_device(op, c.q.device);
  if (st != TRACEA_SUCCESS) return st;
  if (c.lse.device != c.q.device) return fail(TRACEA_INVALID_PARAMS, "%s: operands live on different devices", op);
  for (int i = 0; i < (c.backward ? 7 : 3); ++i)
    if (halves[i]->device != c.q.device) return fail(TRACEA_INVALID_PARAMS, "%s: operands live on different devices", op);
  if ((st = read_lengths(op, "q_lengths", q_lengths, B, c.q.device, c.q_lengths, &c.q_len)) != TRACEA_SUCCESS) return st;
  if ((st = read_lengths(op, "k_lengths", k_lengths, B, c.q.device, c.k_lengths, &c.k_len)) != TRACEA_SUCCESS) return st;
  if (B == 0 || Hq == 0) {
    *nothing = true;
    return Hk == 0 || B == 0 || Sk == 0 ? TRACEA_SUCCESS : fail(TRACEA_INVALID_PARAMS, "%s: no query heads for %lld key heads", op, Hk);
  }
  if (Hk == 0 || Hq % Hk != 0)
    return fail(TRACEA_INVALID_PARAMS, "%s: %lld query heads are not a multiple of %lld key/value heads", op, Hq, Hk);
  if (D < 1 || D > 128) return fail(TRACEA_UNSUPPORTED_CONFIG, "%s: head dim %lld (1 to 128 supported)", op, D);
  const long long G = Hq / Hk;
  // (rows are divided by G with a 32-bit product, rows and keys counted in 32 bits, B * Hk problems are workgroups of a launch)
  if (G * G * (Sq + 128) >= (1ll << 31) || G * (Sq + Sk + 128) >= (1ll << 31) || B * Hk >= kMostBlocks)
    return fail(TRACEA_UNSUPPORTED_CONFIG, "%s: %lld x %lld key/value heads of %lld x %lld queries over %lld keys are more than is supported",
                op, B, Hk, G, Sq, Sk);
  c.scale = params.scale;
  if (c.scale == 0.0f) c.scale = 1.0f / sqrtf((float)D);
  if (!std::isfinite(c.scale)) return fail(TRACEA_INVALID_PARAMS, "%s: scale is not finite", op);
  c.causal = params.causal ? 1 : 0;
  c.stream = (hipStream_t)params.stream;
  return TRACEA_SUCCESS;
}

// (the kernels read the lengths while others of their workgroups write)
bool over_lengths(const Attention &c, const View &result) {
  return (c.q_len != nullptr && may_overlap(result, c.q_lengths)) || (c.k_len != nullptr && may_overlap(result, c.k_lengths));
}

}  // namespace

TraceaStatus dispatch_attention_forward(const TraceaTensorView &q, const TraceaTensorView &k, const TraceaTensorView &v,
                                        const TraceaTensorView *q_lengths, const TraceaTensorView *k_lengths,
                                        TraceaTensorView *o, TraceaTensorView *lse, const TraceaAttentionParams &params) {
  Attention c;
  const char *op = c.op = "tracea_attention_forward";
  TraceaStatus st;
  if ((st = ready(op)) != TRACEA_SUCCESS) return st;
  if (o == nullptr || lse == nullptr) return fail(TRACEA_INVALID_PARAMS, "%s: output view is NULL", op);
  if ((st = read(op, "q", q, 4, &c.q)) != TRACEA_SUCCESS || (st = read(op, "k", k, 4, &c.k)) != TRACEA_SUCCESS ||
      (st = read(op, "v", v, 4, &c.v)) != TRACEA_SUCCESS || (st = read(op, "o", *o, 4, &c.o)) != TRACEA_SUCCESS ||
      (st = read(op, "lse", *lse, 3, &c.lse)) != TRACEA_SUCCESS)
    return st;
  bool nothing;
  if ((st = check_attention(c, params, q_lengths, k_lengths, &nothing)) != TRACEA_SUCCESS || nothing) return st;
  if (folds(c.o) || folds(c.lse)) return overlapping(op, "elements of a result share an address");
  if (may_overlap(c.lse, c.q) || may_overlap(c.lse, c.k) || may_overlap(c.lse, c.v) || may_overlap(c.lse, c.o))
    return overlapping(op, "lse overlaps another tensor");
  if (over_lengths(c, c.o) || over_lengths(c, c.lse)) return overlapping(op, "a result overlaps the lengths");
  std::lock_guard<std::mutex> together(g_launches);
  return run_attention(c, false);
}

TraceaStatus dispatch_attention_backward(const TraceaTensorView &q, const TraceaTensorView &k, const TraceaTensorView &v,
                                         const TraceaTensorView &o, const TraceaTensorView &lse, const TraceaTensorView &d_o,
                                         const TraceaTensorView *q_lengths, const TraceaTensorView *k_lengths,
                                         TraceaTensorView *dq, TraceaTensorView *dk, TraceaTensorView *dv,
                                         const TraceaAttentionParams &params) {
  Attention c;
  const char *op = c.op = "tracea_attention_backward";
  c.backward = true;
  TraceaStatus st;
  if ((st = ready(op)) != TRACEA_SUCCESS) return st;
  if (dq == nullptr || dk == nullptr || dv == nullptr) return fail(TRACEA_INVALID_PARAMS, "%s: output view is NULL", op);
  if ((st = read(op, "q", q, 4, &c.q)) != TRACEA_SUCCESS || (st = read(op, "k", k, 4, &c.k)) != TRACEA_SUCCESS ||
      (st = read(op, "v", v, 4, &c.v)) != TRACEA_SUCCESS || (st = read(op, "o", o, 4, &c.o)) != TRACEA_SUCCESS ||
      (st = read(op, "lse", lse, 3, &c.lse)) != TRACEA_SUCCESS || (st = read(op, "d_o", d_o, 4, &c.d_o)) != TRACEA_SUCCESS ||
      (st = read(op, "dq", *dq, 4, &c.dq)) != TRACEA_SUCCESS || (st = read(op, "dk", *dk, 4, &c.dk)) != TRACEA_SUCCESS ||
      (st = read(op, "dv", *dv, 4, &c.dv)) != TRACEA_SUCCESS)
    return st;
  bool nothing;
  if ((st = check_attention(c, params, q_lengths, k_lengths, &nothing)) != TRACEA_SUCCESS || nothing) return st;
  const View *results[3] = {&c.dq, &c.dk, &c.dv};
  for (int i = 0; i < 3; ++i) {
    if (folds(*results[i])) return overlapping(op, "elements of a result share an address");
    if (may_overlap(*results[i], c.lse)) return overlapping(op, "a result overlaps lse");
    if (over_lengths(c, *results[i])) return overlapping(op, "a result overlaps the lengths");
    for (int j = 0; j < i; ++j)
      if (may_overlap(*results[i], *results[j])) return overlapping(op, "results overlap each other");
  }
  std::lock_guard<std::mutex> together(g_launches);
  return run_attention(c, false);
}

// ---- rotary ---------------------------------------------------------------------------------------------------

TraceaStatus dispatch_rotary(const TraceaTensorView &tq, const TraceaTensorView *tk, const TraceaTensorView &tpos,
                             const TraceaTensorView &tfreq, TraceaTensorView *tq_out, TraceaTensorView *tk_out,
                             const TraceaRotaryParams &params) {
  const char *op = "tracea_rotary";
  TraceaStatus st;
  if ((st = ready(op)) != TRACEA_SUCCESS) return st;
  if (tq_out == nullptr || (tk == nullptr) != (tk_out == nullptr))
    return fail(TRACEA_INVALID_PARAMS, "%s: every operand needs a result, and every result an operand", op);
  View q, k, pos, freq, qo, ko;
  if ((st = read(op, "q", tq, 4, &q)) != TRACEA_SUCCESS || (st = read(op, "q_out", *tq_out, 4, &qo)) != TRACEA_SUCCESS ||
      (st = read(op, "positions", tpos, 3, &pos)) != TRACEA_SUCCESS || (st = read(op, "inv_freq", tfreq, 1, &freq)) != TRACEA_SUCCESS)
    return st;
  const bool two = tk != nullptr;
  if (two && ((st = read(op, "k", *tk, 4, &k)) != TRACEA_SUCCESS || (st = read(op, "k_out", *tk_out, 4, &ko)) != TRACEA_SUCCESS)) return st;
  if (!is_float_type(q.dtype)) return fail(TRACEA_UNSUPPORTED_CONFIG, "%s: f32, f16 or bf16 tensors (got %s)", op, dtype_name(q.dtype));
  if (qo.dtype != q.dtype || (two && (k.dtype != q.dtype || ko.dtype != q.dtype)))
    return fail(TRACEA_UNSUPPORTED_CONFIG, "%s: q, k and their results must share one type", op);
  const long long B = q.shape[0], S = q.shape[2], D = q.shape[3], P = freq.shape[0];
  if (!same_shape(q, qo) || (two && (!same_shape(k, ko) || k.shape[0] != B || k.shape[2] != S || k.shape[3] != D)))
    return fail(TRACEA_INVALID_PARAMS, "%s: q and q_out must be [B,Hq,S,D], k and k_out [B,Hk,S,D]", op);
  if (params.axes < 1 || params.axes > TRACEA_MAX_ROTARY_AXES)
    return fail(TRACEA_INVALID_PARAMS, "%s: %u axes (1 to %d supported)", op, params.axes, TRACEA_MAX_ROTARY_AXES);
  if (pos.dtype != TRACEA_DTYPE_INT32 || (pos.shape[0] != B && pos.shape[0] != 1) || pos.shape[1] != S || pos.shape[2] != (long long)params.axes ||
      (params.axes > 1 && pos.stride[2] != 1))
    return fail(TRACEA_INVALID_PARAMS, "%s: positions must be i32 [B,S,A] or [1,S,A] for the A axes, A contiguous", op);
  if (freq.dtype != TRACEA_DTYPE_FLOAT32 || (P > 1 && freq.stride[0] != 1))
    return fail(TRACEA_INVALID_PARAMS, "%s: inv_freq must be a contiguous f32 vector", op);
  long long sum = 0;
  RotaryArgs a{};
  for (uint32_t i = 0; i < params.axes; ++i) {
    a.first[i] = (int)sum;
    sum += params.sections[i];
  }
  if (sum != P || 2 * P > D)
    return fail(TRACEA_INVALID_PARAMS, "%s: the sections hold %lld pairs, inv_freq %lld, a head dim of %lld at most %lld", op, sum, P, D, D / 2);
  if ((st = check_device(op, q.device)) != TRACEA_SUCCESS) return st;
  const View *all[5] = {&qo, &pos, &freq, two ? &k : &q, two ? &ko : &q};
  for (const View *t : all)
    if (t->device != q.device) return fail(TRACEA_INVALID_PARAMS, "%s: operands live on different devices", op);
  if (B == 0 || S == 0 || D == 0 || q.shape[1] + (two ? k.shape[1] : 0) == 0) return TRACEA_SUCCESS;
  const View *in[2] = {&q, &k}, *out[2] = {&qo, &ko};
  for (int i = 0; i < (two ? 2 : 1); ++i) {
    if ((in[i]->stride[3] != 1 || out[i]->stride[3] != 1) && D > 1)
      return fail(TRACEA_UNSUPPORTED_CONFIG, "%s: the head dimension must be contiguous", op);
    if (folds(*out[i])) return overlapping(op, "elements of a result share an address");
    if (may_overlap(*out[i], pos) || may_overlap(*out[i], freq)) return overlapping(op, "a result overlaps positions or inv_freq");
    for (int j = 0; j < (two ? 2 : 1); ++j)
      if (!(i == j && same_view(*out[i], *in[j])) && may_overlap(*out[i], *in[j]))
        return overlapping(op, "a result overlaps an operand other than its own, or its own in part");
  }
  if (two && may_overlap(qo, ko)) return overlapping(op, "results overlap each other");
  a.q = head_view(q); a.q_out = head_view(qo);
  a.Hq = (int)q.shape[1];
  if (two) {
    a.k = head_view(k); a.k_out = head_view(ko);
    a.Hk = (int)k.shape[1];
  }
  a.positions = (const int *)pos.ptr;
  a.pos_sb = pos.shape[0] == 1 ? 0 : pos.stride[0];
  a.pos_ss = pos.stride[1];
  a.inv_freq = (const float *)freq.ptr;
  a.B = (int)B; a.S = (int)S; a.D = (int)D; a.P = (int)P; a.axes = (int)params.axes;
  a.adjacent = params.adjacent != 0;
  a.inverse = params.inverse != 0;
  const int e = 16 / elem_size(q.dtype);
  a.vec = P % e == 0 && (D - 2 * P) % e == 0;
  for (int i = 0; i < (two ? 2 : 1); ++i)
    for (const View *t : {in[i], out[i]}) {
      if (!aligned(t->ptr, 16)) a.vec = 0;
      for (int d = 0; d < 3; ++d)
        if (t->shape[d] > 1 && t->stride[d] % e != 0) a.vec = 0;
    }
  const long long pieces = a.vec ? (P + D - 2 * P) / e : D - P, heads = a.Hq + a.Hk;
  long long threads = B * S * pieces;
  // Angles are worked out once for the heads of a thread: fewer of them where threads would be few (16 waves per CU).
  const long long want = device_limits().cus * 16 * 64;
  long long groups = (want + threads - 1) / threads;
  groups = groups < 1 ? 1 : groups > heads ? heads : groups;
  // Where the heads of a token are next to each other in memory, at least 8 threads next to each other share them (S24960 H32:8 D128 bf16
  // 98 us; workgroups of 20 heads each 127); where they are a sequence apart, workgroups of at most 6 heads do (98 us; of 20, 106).
  const long long apart = S > 1 ? q.stride[2] : q.stride[0];
  a.beside = 1;
  if (a.Hq > 1 && std::llabs(q.stride[1]) < std::llabs(apart)) {
    a.beside = (int)std::min(heads, std::max(groups, 8ll));
    a.heads_per_group = (int)heads;
    threads *= a.beside;
  } else {
    groups = std::max(groups, (heads + 5) / 6);
    if (heads / groups > 65535) groups = (heads + 65534) / 65535;
    a.heads_per_group = (int)((heads + groups - 1) / groups);
    if ((heads + a.heads_per_group - 1) / a.heads_per_group > 65535) a.heads_per_group = (int)((heads + 65534) / 65535);
  }
  if ((threads + 255) / 256 >= (1ll << 31)) return fail(TRACEA_UNSUPPORTED_CONFIG, "%s: problem too large", op);
  DeviceScope scope(q.device);
  if (scope.err != hipSuccess) return hip_status("hipSetDevice", (int)scope.err);
  return hip_status("rotary launch", launch_rotary(a, q.dtype, (hipStream_t)params.stream));
}

// ---- norm, gate, residual ---------------------------------------------------------------------------------------

namespace {

struct NormCall {
  const char *op;
  long long B, T, C;
  int dtype, device;
};

TraceaStatus read_rows(const NormCall &c, const char *name, const TraceaTensorView *t, RowView *out, View *v) {
  TraceaStatus st = read(c.op, name, *t, 3, v);
  if (st != TRACEA_SUCCESS) return st;
  if (v->dtype != c.dtype) return fail(TRACEA_UNSUPPORTED_CONFIG, "%s: all [B,T,C] tensors must share one type (%s is %s)", c.op, name, dtype_name(v->dtype));
  if (v->shape[0] != c.B || v->shape[1] != c.T || v->shape[2] != c.C)
    return fail(TRACEA_INVALID_PARAMS, "%s: all of x, h, x_out, y and their gradients must share one [B,T,C] shape (%s differs)", c.op, name);
  if (v->device != c.device) return fail(TRACEA_INVALID_PARAMS, "%s: operands live on different devices", c.op);
  if (v->stride[2] != 1 && c.C > 1) return fail(TRACEA_UNSUPPORTED_CONFIG, "%s: the channels must be contiguous (%s)", c.op, name);
  *out = RowView{v->ptr, v->stride[0], v->stride[1]};
  return TRACEA_SUCCESS;
}

TraceaStatus read_vector(const NormCall &c, const char *name, const TraceaTensorView *t, float **out, View *v) {
  if (t == nullptr) return TRACEA_SUCCESS;
  TraceaStatus st = read(c.op, name, *t, 1, v);
  if (st != TRACEA_SUCCESS) return st;
  if (v->dtype != TRACEA_DTYPE_FLOAT32 || v->shape[0] != c.C || (c.C > 1 && v->stride[0] != 1))
    return fail(TRACEA_INVALID_PARAMS, "%s: %s must be a contiguous f32 vector of the %lld channels", c.op, name, c.C);
  if (v->device != c.device) return fail(TRACEA_INVALID_PARAMS, "%s: operands live on different devices", c.op);
  *out = (float *)v->ptr;
  return TRACEA_SUCCESS;
}

// gate and dgate: [G,C], G = 1 or B
TraceaStatus read_gate(const NormCall &c, const char *name, const TraceaTensorView *t, float **out, long long *gates, View *v) {
  if (t == nullptr) return TRACEA_SUCCESS;
  TraceaStatus st = read(c.op, name, *t, 2, v);
  if (st != TRACEA_SUCCESS) return st;
  if (v->dtype != TRACEA_DTYPE_FLOAT32 || v->shape[1] != c.C || (v->shape[0] != 1 && v->shape[0] != c.B) || (c.C > 1 && v->stride[1] != 1) ||
      (v->shape[0] > 1 && v->stride[0] != c.C))
    return fail(TRACEA_INVALID_PARAMS, "%s: %s must be a contiguous f32 tensor [1,C] or [B,C]", c.op, name);
  if (v->device != c.device) return fail(TRACEA_INVALID_PARAMS, "%s: operands live on different devices", c.op);
  *out = (float *)v->ptr;
  *gates = v->shape[0];
  return TRACEA_SUCCESS;
}

TraceaStatus norm_call(NormCall &c, const TraceaTensorView &x, const TraceaNormParams &params) {
  View v;
  TraceaStatus st = read(c.op, "x", x, 3, &v);
  if (st != TRACEA_SUCCESS) return st;
  c.B = v.shape[0]; c.T = v.shape[1]; c.C = v.shape[2];
  c.dtype = v.dtype;
  c.device = v.device;
  if (!is_float_type(c.dtype)) return fail(TRACEA_UNSUPPORTED_CONFIG, "%s: f32, f16 or bf16 tensors (got %s)", c.op, dtype_name(c.dtype));
  if (c.C < 1 || c.C > kNormMaxChannels) return fail(TRACEA_UNSUPPORTED_CONFIG, "%s: %lld channels (1 to %d supported)", c.op, c.C, kNormMaxChannels);
  if (c.B > 65000) return fail(TRACEA_UNSUPPORTED_CONFIG, "%s: more than 65000 batch entries", c.op);
  // (rows are counted in 32 bits, up to the end of the last workgroup's run)
  if (c.T > (1ll << 31) - (1 << 20)) return fail(TRACEA_UNSUPPORTED_CONFIG, "%s: %lld rows (up to 2^31 - 2^20 supported)", c.op, c.T);
  if (!std::isfinite(params.eps) || params.eps < 0.0f || !std::isfinite(params.residual_scale))
    return fail(TRACEA_INVALID_PARAMS, "%s: eps must be finite and not negative, residual_scale finite", c.op);
  return check_device(c.op, c.device);
}

void finish(const NormCall &c, const View *const *tensors, int n, bool backward, const TraceaNormParams &params, NormArgs *a) {
  a->B = (int)c.B; a->T = (int)c.T; a->C = (int)c.C;
  a->eps = params.eps;
  a->scale = params.residual_scale;
  const long long e = 16 / elem_size(c.dtype);
  a->vec = c.C % 8 == 0;
  for (int i = 0; i < n; ++i)
    if (!aligned(tensors[i]->ptr, 16) || (c.B > 1 && tensors[i]->stride[0] % e != 0) || (c.T > 1 && tensors[i]->stride[1] % e != 0)) a->vec = 0;
  for (const float *w : {a->w_post, a->gate, a->w_pre})
    if (!aligned(w, 16)) a->vec = 0;
  a->chunks = norm_chunks(a->B, a->T, a->C, (int)device_limits().cus, backward);
  a->rows_per_chunk = (a->T + a->chunks - 1) / a->chunks;
}

}  // namespace

TraceaStatus dispatch_norm(const TraceaTensorView &x, const TraceaTensorView *h, const TraceaTensorView *w_post,
                           const TraceaTensorView *gate, const TraceaTensorView *w_pre, TraceaTensorView *x_out,
                           TraceaTensorView *y, const TraceaNormParams &params) {
  NormCall c{};
  const char *op = c.op = "tracea_norm_gate_residual";
  TraceaStatus st;
  if ((st = ready(op)) != TRACEA_SUCCESS) return st;
  if ((h != nullptr) != (w_post != nullptr) || (h != nullptr) != (x_out != nullptr) || (gate != nullptr && h == nullptr))
    return fail(TRACEA_INVALID_PARAMS, "%s: h, w_post and x_out go together, and gate needs them", op);
  if ((y != nullptr) != (w_pre != nullptr)) return fail(TRACEA_INVALID_PARAMS, "%s: y and w_pre go together", op);
  if (h == nullptr && y == nullptr) return fail(TRACEA_INVALID_PARAMS, "%s: nothing to compute (neither h nor y)", op);
  if ((st = norm_call(c, x, params)) != TRACEA_SUCCESS) return st;
  NormArgs a{};
  View vx, vh, vo, vy, w1, w2, vg;
  long long gates = 1;
  if ((st = read_rows(c, "x", &x, &a.x, &vx)) != TRACEA_SUCCESS) return st;
  if (h != nullptr && ((st = read_rows(c, "h", h, &a.h, &vh)) != TRACEA_SUCCESS || (st = read_rows(c, "x_out", x_out, &a.x_out, &vo)) != TRACEA_SUCCESS)) return st;
  if (y != nullptr && (st = read_rows(c, "y", y, &a.y, &vy)) != TRACEA_SUCCESS) return st;
  if ((st = read_vector(c, "w_post", w_post, (float **)&a.w_post, &w1)) != TRACEA_SUCCESS ||
      (st = read_vector(c, "w_pre", w_pre, (float **)&a.w_pre, &w2)) != TRACEA_SUCCESS ||
      (st = read_gate(c, "gate", gate, (float **)&a.gate, &gates, &vg)) != TRACEA_SUCCESS)
    return st;
  a.gate_sb = gates == 1 ? 0 : c.C;
  const View *tensors[4];
  int n = 0;
  tensors[n++] = &vx;
  if (h != nullptr) { tensors[n++] = &vh; tensors[n++] = &vo; }
  if (y != nullptr) tensors[n++] = &vy;
  // a result may be x or h as the same view: a thread reads its channels of a row before it writes them
  const View *results[2] = {h != nullptr ? &vo : nullptr, y != nullptr ? &vy : nullptr};
  for (const View *r : results) {
    if (r == nullptr) continue;
    if (folds(*r)) return overlapping(op, "elements of a result share an address");
    if ((!same_view(*r, vx) && may_overlap(*r, vx)) || (h != nullptr && !same_view(*r, vh) && may_overlap(*r, vh)))
      return overlapping(op, "a result overlaps an operand in part");
    if ((w_post != nullptr && may_overlap(*r, w1)) || (w_pre != nullptr && may_overlap(*r, w2)) || (gate != nullptr && may_overlap(*r, vg)))
      return overlapping(op, "a result overlaps a weight");
  }
  if (h != nullptr && y != nullptr && may_overlap(vo, vy)) return overlapping(op, "results overlap each other");
  if (c.B == 0 || c.T == 0) return TRACEA_SUCCESS;
  finish(c, tensors, n, false, params, &a);
  DeviceScope scope(c.device);
  if (scope.err != hipSuccess) return hip_status("hipSetDevice", (int)scope.err);
  return hip_status("norm launch", launch_norm_forward(a, c.dtype, (hipStream_t)params.stream));
}

TraceaStatus dispatch_norm_backward(const TraceaTensorView *dx_out, const TraceaTensorView *dy, const TraceaTensorView &x_out,
                                    const TraceaTensorView *h, const TraceaTensorView *w_post, const TraceaTensorView *gate,
                                    const TraceaTensorView *w_pre, TraceaTensorView *dx, TraceaTensorView *dh,
                                    TraceaTensorView *dw_post, TraceaTensorView *dgate, TraceaTensorView *dw_pre,
                                    const TraceaNormParams &params) {
  NormCall c{};
  const char *op = c.op = "tracea_norm_gate_residual_backward";
  TraceaStatus st;
  if ((st = ready(op)) != TRACEA_SUCCESS) return st;
  if (dx == nullptr) return fail(TRACEA_INVALID_PARAMS, "%s: dx is NULL", op);
  if ((h != nullptr) != (w_post != nullptr) || (h == nullptr && (gate != nullptr || dh != nullptr || dw_post != nullptr)) ||
      (dgate != nullptr && gate == nullptr))
    return fail(TRACEA_INVALID_PARAMS, "%s: h and w_post go together; gate, dh and dw_post need them, dgate needs gate", op);
  if ((dy != nullptr) != (w_pre != nullptr) || (dw_pre != nullptr && dy == nullptr))
    return fail(TRACEA_INVALID_PARAMS, "%s: dy and w_pre go together, dw_pre needs them", op);
  if (h == nullptr && dy == nullptr) return fail(TRACEA_INVALID_PARAMS, "%s: nothing to compute (neither h nor dy)", op);
  if ((st = norm_call(c, x_out, params)) != TRACEA_SUCCESS) return st;
  NormArgs a{};
  View vxo, vh, vdxo, vdy, vdx, vdh, w1, w2, vg, v1, v2, v3;
  const View *tensors[6];
  int n = 0;
  long long gates = 1, dgates = 1;
  if ((st = read_rows(c, "x_out", &x_out, &a.x_out, &vxo)) != TRACEA_SUCCESS || (st = read_rows(c, "dx", dx, &a.dx, &vdx)) != TRACEA_SUCCESS) return st;
  tensors[n++] = &vxo;
  tensors[n++] = &vdx;
  if (h != nullptr) {
    if ((st = read_rows(c, "h", h, &a.h, &vh)) != TRACEA_SUCCESS) return st;
    tensors[n++] = &vh;
  }
  if (dx_out != nullptr) {
    if ((st = read_rows(c, "dx_out", dx_out, &a.dx_out, &vdxo)) != TRACEA_SUCCESS) return st;
    tensors[n++] = &vdxo;
  }
  if (dy != nullptr) {
    if ((st = read_rows(c, "dy", dy, &a.dy, &vdy)) != TRACEA_SUCCESS) return st;
    tensors[n++] = &vdy;
  }
  if (dh != nullptr) {
    if ((st = read_rows(c, "dh", dh, &a.dh, &vdh)) != TRACEA_SUCCESS) return st;
    tensors[n++] = &vdh;
  }
  if ((st = read_vector(c, "w_post", w_post, (float **)&a.w_post, &w1)) != TRACEA_SUCCESS ||
      (st = read_vector(c, "w_pre", w_pre, (float **)&a.w_pre, &w2)) != TRACEA_SUCCESS ||
      (st = read_gate(c, "gate", gate, (float **)&a.gate, &gates, &vg)) != TRACEA_SUCCESS ||
      (st = read_vector(c, "dw_post", dw_post, &a.dw_post, &v1)) != TRACEA_SUCCESS ||
      (st = read_vector(c, "dw_pre", dw_pre, &a.dw_pre, &v2)) != TRACEA_SUCCESS ||
      (st = read_gate(c, "dgate", dgate, &a.dgate, &dgates, &v3)) != TRACEA_SUCCESS)
    return st;
  if (dgate != nullptr && dgates != gates) return fail(TRACEA_INVALID_PARAMS, "%s: dgate must have gate's shape", op);
  a.gate_sb = gates == 1 ? 0 : c.C;
  const View *rows[2] = {&vdx, dh != nullptr ? &vdh : nullptr};
  const View *sums[3] = {dw_post != nullptr ? &v1 : nullptr, dw_pre != nullptr ? &v2 : nullptr, dgate != nullptr ? &v3 : nullptr};
  const View *reads[7] = {&vxo, h != nullptr ? &vh : nullptr, dx_out != nullptr ? &vdxo : nullptr, dy != nullptr ? &vdy : nullptr,
                          w_post != nullptr ? &w1 : nullptr, w_pre != nullptr ? &w2 : nullptr, gate != nullptr ? &vg : nullptr};
  // dx may be dx_out or dy, dh may be h, as the same view: a thread reads its channels of a row before it writes them
  for (int i = 0; i < 5; ++i) {
    const View *r = i < 2 ? rows[i] : sums[i - 2];
    if (r == nullptr) continue;
    if (folds(*r)) return overlapping(op, "elements of a result share an address");
    for (int j = 0; j < 7; ++j) {
      if (reads[j] == nullptr || (i < 2 && j < 4 && same_view(*r, *reads[j]))) continue;
      if (may_overlap(*r, *reads[j])) return overlapping(op, "a result overlaps an operand (in part)");
    }
    for (int j = 0; j < i; ++j) {
      const View *o = j < 2 ? rows[j] : sums[j - 2];
      if (o != nullptr && may_overlap(*r, *o)) return overlapping(op, "results overlap each other");
    }
  }
  DeviceScope scope(c.device);
  if (scope.err != hipSuccess) return hip_status("hipSetDevice", (int)scope.err);
  hipStream_t stream = (hipStream_t)params.stream;
  const bool columns = dw_post != nullptr || dgate != nullptr || dw_pre != nullptr;
  if ((c.B == 0 || c.T == 0) && !columns) return TRACEA_SUCCESS;
  if (c.B == 0) {  // (no batch entry: sums over one of no rows, without the gates that no entry has)
    c.B = 1;
    c.T = 0;
    if (gates == 0) {
      a.gate = a.dgate = nullptr;
      a.gate_sb = 0;
    }
  }
  finish(c, tensors, n, true, params, &a);
  std::lock_guard<std::mutex> together(g_launches);
  if (columns) {
    a.partial = (float *)train_scratch(c.device, stream, (size_t)2 * a.B * a.chunks * a.C * 4);
    if (a.partial == nullptr)
      return fail(TRACEA_UNSUPPORTED_CONFIG, "%s: no workspace can be had (a stream under capture that made no such call before, or out of "
                                             "memory)", op);
  }
  return hip_status("norm backward launch", launch_norm_backward(a, c.dtype, stream));
}

}  // namespace tracea_amd
