// Argument checks and launches of the operators over a key/value cache: norms of heads with rotary positions, appending to pages, attention
// over them.  Status codes as in dispatch.cpp.
#include <cmath>

#include "../cache.hpp"
#include "operands.hpp"

namespace tracea_amd {

namespace {

TraceaStatus other_device(const char *op) { return fail(TRACEA_INVALID_PARAMS, "%s: operands live on different devices", op); }

// The pairs that positions turn, as tracea_rotary has them; inv_freq null: none.  `own`: positions may be left out (the caller has its own).
struct Rotation {
  View positions, freq;
  const int *pos = nullptr;
  long long pos_sb = 0, pos_ss = 0;
  const float *inv_freq = nullptr;
  int P = 0, axes = 0;
  int first[TRACEA_MAX_ROTARY_AXES] = {0, 0, 0, 0};
};
TraceaStatus read_rotation(const char *op, const TraceaTensorView *tpos, const TraceaTensorView *tfreq, uint32_t axes, const uint32_t *sections,
                           long long B, long long S, long long D, int device, bool own, Rotation *r) {
  if (tfreq == nullptr) {
    if (tpos != nullptr || axes != 0)
      return fail(TRACEA_INVALID_PARAMS, "%s: positions and sections need inv_freq", op);
    return TRACEA_SUCCESS;
  }
  if (tpos == nullptr && !own) return fail(TRACEA_INVALID_PARAMS, "%s: inv_freq needs positions", op);
  if (axes < 1 || axes > TRACEA_MAX_ROTARY_AXES)
    return fail(TRACEA_INVALID_PARAMS, "%s: %u axes (1 to %d supported)", op, axes, TRACEA_MAX_ROTARY_AXES);
  if (tpos == nullptr && axes != 1) return fail(TRACEA_INVALID_PARAMS, "%s: %u axes need positions", op, axes);
  TraceaStatus st;
  if ((st = read(op, "inv_freq", *tfreq, 1, &r->freq)) != TRACEA_SUCCESS) return st;
  const long long P = r->freq.shape[0];
  if (r->freq.dtype != TRACEA_DTYPE_FLOAT32 || (P > 1 && r->freq.stride[0] != 1))
    return fail(TRACEA_INVALID_PARAMS, "%s: inv_freq must be a contiguous f32 vector", op);
  if (r->freq.device != device) return other_device(op);
  if (tpos != nullptr) {
    const View &v = r->positions;
    if ((st = read(op, "positions", *tpos, 3, &r->positions)) != TRACEA_SUCCESS) return st;
    if (v.dtype != TRACEA_DTYPE_INT32 || (v.shape[0] != B && v.shape[0] != 1) || v.shape[1] != S || v.shape[2] != (long long)axes ||
        (axes > 1 && v.stride[2] != 1))
      return fail(TRACEA_INVALID_PARAMS, "%s: positions must be i32 [B,S,A] or [1,S,A] for the A axes, A contiguous", op);
    if (v.device != device) return other_device(op);
    r->pos = (const int *)v.ptr;
    r->pos_sb = v.shape[0] == 1 ? 0 : v.stride[0];
    r->pos_ss = v.stride[1];
  }
  long long sum = 0;
  for (uint32_t i = 0; i < axes; ++i) {
    r->first[i] = (int)std::min(sum, P);
    sum += sections[i];
  }
  if (sum != P || 2 * P > D)
    return fail(TRACEA_INVALID_PARAMS, "%s: the sections hold %lld pairs, inv_freq %lld, a head dim of %lld at most %lld", op, sum, P, D, D / 2);
  r->inv_freq = (const float *)r->freq.ptr;
  r->P = (int)P;
  r->axes = (int)axes;
  return TRACEA_SUCCESS;
}
bool over_rotation(const Rotation &r, const View &result) {
  return (r.pos != nullptr && may_overlap(result, r.positions)) || (r.inv_freq != nullptr && may_overlap(result, r.freq));
}
template <typename Args>
void set_rotation(const Rotation &r, Args *a) {
  a->positions = r.pos;
  a->pos_sb = r.pos_sb;
  a->pos_ss = r.pos_ss;
  a->inv_freq = r.inv_freq;
  a->P = r.P;
  a->axes = r.axes;
  for (int i = 0; i < TRACEA_MAX_ROTARY_AXES; ++i) a->first[i] = r.first[i];
}

// Whether every row begins on `bytes`.
bool rows_on(const View &t, size_t bytes) {
  if (!aligned(t.ptr, bytes)) return false;
  const long long e = (long long)bytes / elem_size(t.dtype);
  for (int i = 0; i + 1 < t.rank; ++i)
    if (t.shape[i] > 1 && t.stride[i] % e != 0) return false;
  return true;
}
bool columns_apart(const View &t) { return t.shape[t.rank - 1] > 1 && t.stride[t.rank - 1] != 1; }

// [B] i32 on `device`
TraceaStatus read_counts(const char *op, const char *name, const TraceaTensorView *t, long long B, int device, View *v, const int **out) {
  if (t == nullptr) return TRACEA_SUCCESS;
  TraceaStatus st = read(op, name, *t, 1, v);
  if (st != TRACEA_SUCCESS) return st;
  if (v->dtype != TRACEA_DTYPE_INT32 || v->shape[0] != B || (B > 1 && v->stride[0] != 1))
    return fail(TRACEA_INVALID_PARAMS, "%s: %s must be a contiguous i32 tensor of %lld entries, one per sequence", op, name, B);
  if (v->device != device) return other_device(op);
  *out = (const int *)v->ptr;
  return TRACEA_SUCCESS;
}

// The two caches with their scales and the table of their pages.
struct Cache {
  View k, v, ks, vs, table;
  bool e4m3 = false;
  PageView kp{}, vp{};
  ScaleView ksp{}, vsp{};
  PageTable pages{};
};
TraceaStatus read_cache(const char *op, const TraceaTensorView &tk, const TraceaTensorView &tv, const TraceaTensorView *tks,
                        const TraceaTensorView *tvs, const TraceaTensorView &ttable, int dtype, int device, long long B, long long Hk, long long D,
                        Cache *c) {
  TraceaStatus st;
  if ((st = read(op, "k_cache", tk, 4, &c->k)) != TRACEA_SUCCESS || (st = read(op, "v_cache", tv, 4, &c->v)) != TRACEA_SUCCESS ||
      (st = read(op, "page_table", ttable, 2, &c->table)) != TRACEA_SUCCESS)
    return st;
  c->e4m3 = c->k.dtype == TRACEA_DTYPE_FLOAT8_E4M3;
  if (c->k.dtype != c->v.dtype || (!c->e4m3 && c->k.dtype != dtype))
    return fail(TRACEA_UNSUPPORTED_CONFIG, "%s: both caches must be of the operands' type or e4m3 (got %s and %s)", op, dtype_name(c->k.dtype),
                dtype_name(c->v.dtype));
  if (c->e4m3 != (tks != nullptr) || c->e4m3 != (tvs != nullptr))
    return fail(TRACEA_INVALID_PARAMS, "%s: k_scale and v_scale go with caches of 8 bits", op);
  const long long N = c->k.shape[0], P = c->k.shape[2];
  if (!same_shape(c->k, c->v) || c->k.shape[1] != Hk || c->k.shape[3] != D)
    return fail(TRACEA_INVALID_PARAMS, "%s: k_cache and v_cache must be [N,Hk,P,D] with the keys' heads and head dim", op);
  if (P < 16 || P % 16 != 0) return fail(TRACEA_UNSUPPORTED_CONFIG, "%s: pages of %lld tokens (a multiple of 16 supported)", op, P);
  if (D % 8 != 0) return fail(TRACEA_UNSUPPORTED_CONFIG, "%s: head dim %lld (a multiple of 8 supported)", op, D);
  if (c->table.dtype != TRACEA_DTYPE_INT32 || c->table.shape[0] != B || (c->table.shape[1] > 1 && c->table.stride[1] != 1))
    return fail(TRACEA_INVALID_PARAMS, "%s: page_table must be i32 [B,M], M contiguous", op);
  // (places and keys are counted in 32 bits, up to the end of the last step)
  const long long M = c->table.shape[1];
  if (M * P > (1ll << 31) - (1 << 16) || M * P * P >= (1ll << 40))
    return fail(TRACEA_UNSUPPORTED_CONFIG, "%s: %lld pages of %lld tokens a sequence (M P up to 2^31 - 2^16, M P P below 2^40 supported)", op, M, P);
  const View *of_device[3] = {&c->k, &c->v, &c->table};
  for (const View *t : of_device)
    if (t->device != device) return other_device(op);
  const long long e = elem_size(c->k.dtype);
  for (const View *t : {&c->k, &c->v}) {
    if (columns_apart(*t)) return fail(TRACEA_UNSUPPORTED_CONFIG, "%s: the head dimension of a cache must be contiguous", op);
    for (int i = 0; i < 3; ++i)
      if (t->shape[i] > 1 && (t->stride[i] % 8 != 0 || t->stride[i] < 0))
        return fail(TRACEA_UNSUPPORTED_CONFIG, "%s: strides of a cache must be multiples of 8 elements, not negative", op);
    if (count_of(*t) > 0 && !aligned(t->ptr, (size_t)(8 * e))) return fail(TRACEA_UNSUPPORTED_CONFIG, "%s: a cache must begin on %lld bytes", op, 8 * e);
    // (offsets within 16 tokens of a page are 32-bit)
    if (t->stride[2] * 16 * e >= (1ll << 31)) return fail(TRACEA_UNSUPPORTED_CONFIG, "%s: tokens of a cache 2^27 bytes apart", op);
  }
  c->kp = PageView{(unsigned char *)c->k.ptr, c->k.stride[0] * e, c->k.stride[1] * e, c->k.stride[2] * e};
  c->vp = PageView{(unsigned char *)c->v.ptr, c->v.stride[0] * e, c->v.stride[1] * e, c->v.stride[2] * e};
  if (c->e4m3) {
    if ((st = read(op, "k_scale", *tks, 2, &c->ks)) != TRACEA_SUCCESS || (st = read(op, "v_scale", *tvs, 2, &c->vs)) != TRACEA_SUCCESS) return st;
    for (const View *t : {&c->ks, &c->vs}) {
      if (t->dtype != TRACEA_DTYPE_FLOAT32 || t->shape[0] != N || t->shape[1] != Hk)
        return fail(TRACEA_INVALID_PARAMS, "%s: k_scale and v_scale must be f32 [N,Hk]", op);
      if (t->device != device) return other_device(op);
    }
    c->ksp = ScaleView{(float *)c->ks.ptr, c->ks.stride[0], c->ks.stride[1]};
    c->vsp = ScaleView{(float *)c->vs.ptr, c->vs.stride[0], c->vs.stride[1]};
  }
  c->pages = PageTable{(const int *)c->table.ptr, c->table.stride[0], (int)M, (int)N, (int)P};
  return TRACEA_SUCCESS;
}

// Whether problems (blocks of up to 32 rows) of up to `most` steps share their steps out.  Unshared, a workgroup walks its problem at 0.75 to
// 1.1 us a step, more slowly the more walk beside it; shared, the lengths are worked through and parts are joined by a second launch, 4.2 us more
// and up to 1.8 where many shares begin inside a problem; then all workgroups read at what the caches' bytes allow.  us unshared / shared, one
// query, Hk 8, D128, lengths from a quarter of the longest up, 8 bits: B1 512 keys 8.5 / 9.8, 800 10.5 / 10.2; B16 800 12.6 / 13.6, 2000 21.3 / 17.4; B30 2000
// 22.0 / 27.5; B32 4096 51 / 46; B100 4096 121 / 118; 16 bits: B4 1000 13.7 / 10.5; B16 1200 18.6 / 21.6, 2000 26 / 21; B12 4096 49 / 28; B48 4096 118 / 101; 20 rows,
// Hk 4, D96, 16 bits: B16 700 14.1 / 14.4, 1000 16.4 / 14.6; B160 2000 73 / 87.
bool shares_pay(long long problems, long long most, bool e4m3, double width, int rows) {
  if (most <= 2 || problems * most >= (1ll << 30) || problems > 65535) return false;
  const double n = (double)problems, more = rows > 16 ? 1.1 : 1.0;
  const double alone = 5.5 * more + most * std::max(more * (e4m3 ? 0.75 + 0.002 * n : 1.0 + 0.004 * n), (e4m3 ? 5.0e-3 : 8.2e-3) * width * n);
  const double shared = 9.7 + 1.8 * std::min(1.0, n / 128) + (rows > 16 ? 1.15 : 1.0) * most * (e4m3 ? 4.1e-3 : 7.0e-3) * width * n;
  return alone > shared;
}

// Parts of the steps (tiles of 64 keys) of blocks of 128 rows, by the least of this estimate (us).  A workgroup alone on its CU takes 1.8 us a
// tile, two 2.5 each; parts cost a launch that joins them and their way through memory, 66 KB each.  us, one part / best, 8 heads, D128
// e4m3: B1 32 queries over 8192 keys 251 / 31 (32 parts), B4 128 queries over 4096 132 / 63 (4), over 512 24 / 24 (1), B16 32 over 2048 74 / 46 (4).
int plan_tiles(long long problems, long long most, bool e4m3, double width, long long cus) {
  int best = 1;
  double least = 1e300;
  for (int parts : {1, 2, 3, 4, 6, 8, 12, 16, 24, 32}) {
    if (parts > 1 && (parts > most || problems * parts > 4 * cus || problems > 65535)) break;
    const double n = (double)(problems * parts), walk = (double)((most + parts - 1) / parts);
    const double tile = (e4m3 ? 1.0 : 0.85) * (0.3 + 0.7 * width) * std::max(1.8, n > cus ? 2.5 * std::ceil(n / (2.0 * cus)) : 0.0);
    const double time = walk * tile + (parts > 1 ? 4.5 + 0.035 * width * n : 0.0);
    if (time < least) {
      least = time;
      best = parts;
    }
  }
  return best;
}

}  // namespace

// ---- norms of heads with rotary positions ---------------------------------------------------------------------

namespace {

struct QkNorm {
  const char *op;
  long long B, S, D;
  int dtype, device, n;  // n: tensors, 1 or 2
};
TraceaStatus read_heads(const QkNorm &c, const char *name, const TraceaTensorView &t, const View *like, View *v) {
  TraceaStatus st = read(c.op, name, t, 4, v);
  if (st != TRACEA_SUCCESS) return st;
  if (v->dtype != c.dtype) return fail(TRACEA_UNSUPPORTED_CONFIG, "%s: all [B,H,S,D] tensors must share one type (%s is %s)", c.op, name, dtype_name(v->dtype));
  if (v->shape[0] != c.B || v->shape[2] != c.S || v->shape[3] != c.D || (like != nullptr && !same_shape(*v, *like)))
    return fail(TRACEA_INVALID_PARAMS, "%s: q and its results must be [B,Hq,S,D], k and its results [B,Hk,S,D] (%s differs)", c.op, name);
  if (v->device != c.device) return other_device(c.op);
  if (columns_apart(*v)) return fail(TRACEA_UNSUPPORTED_CONFIG, "%s: the head dimension must be contiguous (%s)", c.op, name);
  return TRACEA_SUCCESS;
}
TraceaStatus read_weight(const QkNorm &c, const char *name, const TraceaTensorView *t, float **out, View *v) {
  if (t == nullptr) return TRACEA_SUCCESS;
  TraceaStatus st = read(c.op, name, *t, 1, v);
  if (st != TRACEA_SUCCESS) return st;
  if (v->dtype != TRACEA_DTYPE_FLOAT32 || v->shape[0] != c.D || (c.D > 1 && v->stride[0] != 1))
    return fail(TRACEA_INVALID_PARAMS, "%s: %s must be a contiguous f32 vector of the head dim, %lld", c.op, name, c.D);
  if (v->device != c.device) return other_device(c.op);
  *out = (float *)v->ptr;
  return TRACEA_SUCCESS;
}
TraceaStatus qk_norm_call(const TraceaTensorView &q, bool two, const TraceaQkNormParams &params, QkNorm *c, View *v) {
  TraceaStatus st;
  if ((st = read(c->op, "q", q, 4, v)) != TRACEA_SUCCESS) return st;
  c->B = v->shape[0]; c->S = v->shape[2]; c->D = v->shape[3];
  c->dtype = v->dtype;
  c->device = v->device;
  c->n = two ? 2 : 1;
  if (!is_float_type(c->dtype)) return fail(TRACEA_UNSUPPORTED_CONFIG, "%s: f32, f16 or bf16 tensors (got %s)", c->op, dtype_name(c->dtype));
  if (c->D < 1 || c->D > kQkNormMaxDim) return fail(TRACEA_UNSUPPORTED_CONFIG, "%s: head dim %lld (1 to %d supported)", c->op, c->D, kQkNormMaxDim);
  if (!std::isfinite(params.eps) || params.eps < 0.0f) return fail(TRACEA_INVALID_PARAMS, "%s: eps must be finite and not negative", c->op);
  if (columns_apart(*v)) return fail(TRACEA_UNSUPPORTED_CONFIG, "%s: the head dimension must be contiguous (q)", c->op);
  return check_device(c->op, c->device);
}
void set_qk_norm(const QkNorm &c, const Rotation &r, const View *const *tensors, int n, bool backward, const TraceaQkNormParams &params, QkNormArgs *a) {
  a->B = (int)c.B; a->S = (int)c.S; a->D = (int)c.D;
  set_rotation(r, a);
  a->adjacent = params.adjacent != 0;
  a->eps = params.eps;
  a->inv_d = 1.0f / (float)c.D;
  // Pieces of 16 bytes, or of 8 or 4 where pairs, columns that are not turned (they go two pieces to a thread), strides or addresses do not go into
  // them; else single elements.  S24960 H32:8 bf16, D80 of which 40 turned (8 bytes) 84 us, D40 of which 20 (4 bytes) 74; one by one 371, 351.
  const int size = elem_size(c.dtype);
  for (int e = 16 / size; e >= 2 && a->vec == 0; e /= 2) {
    a->vec = a->P % e == 0 && (c.D - 2 * a->P) % (2 * e) == 0 && c.D / (2 * e) <= 64 ? e : 0;
    for (int i = 0; i < n; ++i)
      if (!rows_on(*tensors[i], (size_t)(e * size))) a->vec = 0;
  }
  a->lanes = 64;
  if (a->vec)
    while (a->lanes * a->vec >= c.D && a->lanes > 1) a->lanes /= 2;
  const long long heads = a->H[0] + a->H[1], tokens = c.B * c.S, groups = 256 / a->lanes;
  // Lane groups that share a token's angles take its heads in turn: as many as fill the device with 8 waves a CU where tokens are few; else,
  // where heads lie side by side, a group for 4 heads forward, 8 at most (pieces next to each other: S24960 D128 bf16, 40 heads by 8 / 4 / 2 groups 99 /
  // 104 / 120 us, 24 by 8 / 6 / 2 69 / 62 / 71, 8 by 8 / 2 40 / 23) and 2 backward, where angles cost more, being worked out for queries and keys apart (4 x
  // 2048 tokens of 40 heads by 2 / 4 65 / 70 us, of 8 20 / 25); where they are a sequence apart, one.
  const long long want = ((long long)device_limits().cus * 8 * (64 / a->lanes) + tokens - 1) / std::max(1ll, tokens);
  const bool side_by_side = a->H[0] > 1 && std::llabs(a->x[0].sh) < std::llabs(c.S > 1 ? a->x[0].ss : a->x[0].sb);
  a->beside = (int)std::max(1ll, std::min(heads, std::max(want, !side_by_side ? 1ll : backward ? 2ll : std::min(8ll, heads / 4))));
  a->blocks = (int)std::max(1ll, std::min((long long)device_limits().cus * kQkNormRuns, (tokens * a->beside + groups - 1) / groups));
}

}  // namespace

TraceaStatus dispatch_qk_norm(const TraceaTensorView &tq, const TraceaTensorView *tk, const TraceaTensorView *q_weight,
                              const TraceaTensorView *k_weight, const TraceaTensorView *positions, const TraceaTensorView *inv_freq,
                              TraceaTensorView *tq_out, TraceaTensorView *tk_out, const TraceaQkNormParams &params) {
  QkNorm c{};
  const char *op = c.op = "tracea_qk_norm_rotary";
  TraceaStatus st;
  if ((st = ready(op)) != TRACEA_SUCCESS) return st;
  if (tq_out == nullptr || (tk == nullptr) != (tk_out == nullptr) || (k_weight != nullptr && tk == nullptr))
    return fail(TRACEA_INVALID_PARAMS, "%s: every operand needs a result, every result and weight an operand", op);
  View x[2], out[2], w[2];
  QkNormArgs a{};
  Rotation r;
  if ((st = qk_norm_call(tq, tk != nullptr, params, &c, &x[0])) != TRACEA_SUCCESS || (st = read_heads(c, "q_out", *tq_out, &x[0], &out[0])) != TRACEA_SUCCESS ||
      (st = read_weight(c, "q_weight", q_weight, (float **)&a.w[0], &w[0])) != TRACEA_SUCCESS ||
      (st = read_weight(c, "k_weight", k_weight, (float **)&a.w[1], &w[1])) != TRACEA_SUCCESS)
    return st;
  if (c.n == 2 && ((st = read_heads(c, "k", *tk, nullptr, &x[1])) != TRACEA_SUCCESS || (st = read_heads(c, "k_out", *tk_out, &x[1], &out[1])) != TRACEA_SUCCESS)) return st;
  if ((st = read_rotation(op, positions, inv_freq, params.axes, params.sections, c.B, c.S, c.D, c.device, false, &r)) != TRACEA_SUCCESS) return st;
  if (c.B == 0 || c.S == 0 || x[0].shape[1] + (c.n == 2 ? x[1].shape[1] : 0) == 0) return TRACEA_SUCCESS;
  const View *tensors[4];
  int n = 0;
  for (int i = 0; i < c.n; ++i) {
    if (folds(out[i])) return overlapping(op, "elements of a result share an address");
    if (over_rotation(r, out[i])) return overlapping(op, "a result overlaps positions or inv_freq");
    for (int j = 0; j < c.n; ++j) {
      if (!(i == j && same_view(out[i], x[j])) && may_overlap(out[i], x[j]))
        return overlapping(op, "a result overlaps an operand other than its own, or its own in part");
      if (a.w[j] != nullptr && may_overlap(out[i], w[j])) return overlapping(op, "a result overlaps a weight");
    }
    a.x[i] = head_view(x[i]);
    a.out[i] = head_view(out[i]);
    a.H[i] = (int)x[i].shape[1];
    tensors[n++] = &x[i];
    tensors[n++] = &out[i];
  }
  if (c.n == 2 && may_overlap(out[0], out[1])) return overlapping(op, "results overlap each other");
  set_qk_norm(c, r, tensors, n, false, params, &a);
  if (c.B * c.S * a.beside >= (1ll << 40)) return fail(TRACEA_UNSUPPORTED_CONFIG, "%s: problem too large", op);
  DeviceScope scope(c.device);
  if (scope.err != hipSuccess) return hip_status("hipSetDevice", (int)scope.err);
  return hip_status("qk norm launch", launch_qk_norm_forward(a, c.dtype, (hipStream_t)params.stream));
}

TraceaStatus dispatch_qk_norm_backward(const TraceaTensorView &tdq_out, const TraceaTensorView *tdk_out, const TraceaTensorView &tq,
                                       const TraceaTensorView *tk, const TraceaTensorView *q_weight, const TraceaTensorView *k_weight,
                                       const TraceaTensorView *positions, const TraceaTensorView *inv_freq, TraceaTensorView *tdq,
                                       TraceaTensorView *tdk, TraceaTensorView *dq_weight, TraceaTensorView *dk_weight,
                                       const TraceaQkNormParams &params) {
  QkNorm c{};
  const char *op = c.op = "tracea_qk_norm_rotary_backward";
  TraceaStatus st;
  if ((st = ready(op)) != TRACEA_SUCCESS) return st;
  if (tdq == nullptr || (tk == nullptr) != (tdk == nullptr) || (tk == nullptr) != (tdk_out == nullptr) || (k_weight != nullptr && tk == nullptr))
    return fail(TRACEA_INVALID_PARAMS, "%s: dk_out, k and dk go together, q needs dq_out and dq, k_weight needs k", op);
  if ((dq_weight != nullptr && q_weight == nullptr) || (dk_weight != nullptr && k_weight == nullptr))
    return fail(TRACEA_INVALID_PARAMS, "%s: the gradient of a weight needs the weight", op);
  View x[2], out[2], dout[2], w[2], dw[2];
  QkNormArgs a{};
  Rotation r;
  if ((st = qk_norm_call(tq, tk != nullptr, params, &c, &x[0])) != TRACEA_SUCCESS || (st = read_heads(c, "dq", *tdq, &x[0], &out[0])) != TRACEA_SUCCESS ||
      (st = read_heads(c, "dq_out", tdq_out, &x[0], &dout[0])) != TRACEA_SUCCESS ||
      (st = read_weight(c, "q_weight", q_weight, (float **)&a.w[0], &w[0])) != TRACEA_SUCCESS ||
      (st = read_weight(c, "k_weight", k_weight, (float **)&a.w[1], &w[1])) != TRACEA_SUCCESS ||
      (st = read_weight(c, "dq_weight", dq_weight, &a.dw[0], &dw[0])) != TRACEA_SUCCESS ||
      (st = read_weight(c, "dk_weight", dk_weight, &a.dw[1], &dw[1])) != TRACEA_SUCCESS)
    return st;
  if (c.n == 2 && ((st = read_heads(c, "k", *tk, nullptr, &x[1])) != TRACEA_SUCCESS || (st = read_heads(c, "dk", *tdk, &x[1], &out[1])) != TRACEA_SUCCESS ||
                   (st = read_heads(c, "dk_out", *tdk_out, &x[1], &dout[1])) != TRACEA_SUCCESS))
    return st;
  if ((st = read_rotation(op, positions, inv_freq, params.axes, params.sections, c.B, c.S, c.D, c.device, false, &r)) != TRACEA_SUCCESS) return st;
  const View *tensors[6], *results[4], *reads[6];
  int n = 0, n_results = 0, n_reads = 0;
  for (int i = 0; i < c.n; ++i) {
    a.x[i] = head_view(x[i]);
    a.out[i] = head_view(out[i]);
    a.dout[i] = head_view(dout[i]);
    a.H[i] = (int)x[i].shape[1];
    tensors[n++] = &x[i];
    tensors[n++] = &out[i];
    tensors[n++] = &dout[i];
    results[n_results++] = &out[i];
    reads[n_reads++] = &x[i];
    reads[n_reads++] = &dout[i];
    if (a.w[i] != nullptr) reads[n_reads++] = &w[i];
  }
  for (int i = 0; i < 2; ++i)
    if (a.dw[i] != nullptr) results[n_results++] = &dw[i];
  for (int i = 0; i < n_results; ++i) {
    if (folds(*results[i])) return overlapping(op, "elements of a result share an address");
    if (over_rotation(r, *results[i])) return overlapping(op, "a result overlaps positions or inv_freq");
    for (int j = 0; j < n_reads; ++j) {
      // dq may be q or dq_out: a row is read whole before it is written
      const bool own = i < c.n && (reads[j] == &x[i] || reads[j] == &dout[i]) && same_view(*results[i], *reads[j]);
      if (!own && may_overlap(*results[i], *reads[j])) return overlapping(op, "a result overlaps an operand other than its own, or its own in part");
    }
    for (int j = 0; j < i; ++j)
      if (may_overlap(*results[i], *results[j])) return overlapping(op, "results overlap each other");
  }
  const bool weights = a.dw[0] != nullptr || a.dw[1] != nullptr;
  const bool nothing = c.B == 0 || c.S == 0 || a.H[0] + a.H[1] == 0;
  if (nothing && !weights) return TRACEA_SUCCESS;
  if (nothing) {  // (the weights' gradients are sums over no rows)
    a.H[0] = a.H[1] = 0;
    c.B = c.S = 1;
  }
  set_qk_norm(c, r, tensors, n, true, params, &a);
  if (nothing) a.positions = nullptr;
  DeviceScope scope(c.device);
  if (scope.err != hipSuccess) return hip_status("hipSetDevice", (int)scope.err);
  hipStream_t stream = (hipStream_t)params.stream;
  std::lock_guard<std::mutex> together(g_launches);
  if (weights) {
    a.partial = (float *)train_scratch(c.device, stream, (size_t)2 * a.blocks * c.D * 4);
    if (a.partial == nullptr)
      return fail(TRACEA_UNSUPPORTED_CONFIG, "%s: no workspace can be had (a stream under capture that made no such call before, or out of "
                                             "memory)", op);
  }
  return hip_status("qk norm backward launch", launch_qk_norm_backward(a, c.dtype, stream));
}

// ---- appending to a cache ---------------------------------------------------------------------------------------

TraceaStatus dispatch_cache_append(const TraceaTensorView &tk, const TraceaTensorView &tv, const TraceaTensorView *tq,
                                   TraceaTensorView *k_cache, TraceaTensorView *v_cache, TraceaTensorView *k_scale,
                                   TraceaTensorView *v_scale, const TraceaTensorView &page_table, const TraceaTensorView &tstarts,
                                   const TraceaTensorView *tlengths, const TraceaTensorView *positions, const TraceaTensorView *inv_freq,
                                   TraceaTensorView *tq_out, const TraceaCacheAppendParams &params) {
  const char *op = "tracea_cache_append";
  TraceaStatus st;
  if ((st = ready(op)) != TRACEA_SUCCESS) return st;
  if (k_cache == nullptr || v_cache == nullptr) return fail(TRACEA_INVALID_PARAMS, "%s: a cache is NULL", op);
  if ((tq == nullptr) != (tq_out == nullptr)) return fail(TRACEA_INVALID_PARAMS, "%s: q and q_out go together", op);
  View k, v, q, qo, starts, lengths;
  CacheAppendArgs a{};
  if ((st = read(op, "k", tk, 4, &k)) != TRACEA_SUCCESS || (st = read(op, "v", tv, 4, &v)) != TRACEA_SUCCESS ||
      (tq != nullptr && ((st = read(op, "q", *tq, 4, &q)) != TRACEA_SUCCESS || (st = read(op, "q_out", *tq_out, 4, &qo)) != TRACEA_SUCCESS)))
    return st;
  if (!is_half(k.dtype)) return fail(TRACEA_UNSUPPORTED_CONFIG, "%s: f16 or bf16 tensors (got %s)", op, dtype_name(k.dtype));
  if (v.dtype != k.dtype || (tq != nullptr && (q.dtype != k.dtype || qo.dtype != k.dtype)))
    return fail(TRACEA_UNSUPPORTED_CONFIG, "%s: q, q_out, k and v must share one type, f16 or bf16", op);
  const long long B = k.shape[0], Hk = k.shape[1], T = k.shape[2], D = k.shape[3];
  if (!same_shape(k, v) || (tq != nullptr && (!same_shape(q, qo) || q.shape[0] != B || q.shape[2] != T || q.shape[3] != D)))
    return fail(TRACEA_INVALID_PARAMS, "%s: k and v must be [B,Hk,T,D], q and q_out [B,Hq,T,D]", op);
  const int device = k.device;
  if ((st = check_device(op, device)) != TRACEA_SUCCESS) return st;
  const View *operands[4] = {&k, &v, tq != nullptr ? &q : &k, tq != nullptr ? &qo : &k};
  for (const View *t : operands) {
    if (t->device != device) return other_device(op);
    if (columns_apart(*t)) return fail(TRACEA_UNSUPPORTED_CONFIG, "%s: the head dimension must be contiguous", op);
  }
  if (D < 1 || D > 512) return fail(TRACEA_UNSUPPORTED_CONFIG, "%s: head dim %lld (up to 512 supported)", op, D);
  Cache c;
  Rotation r;
  if ((st = read_cache(op, *k_cache, *v_cache, k_scale, v_scale, page_table, k.dtype, device, B, Hk, D, &c)) != TRACEA_SUCCESS ||
      (st = read_counts(op, "starts", &tstarts, B, device, &starts, &a.starts)) != TRACEA_SUCCESS ||
      (st = read_counts(op, "lengths", tlengths, B, device, &lengths, &a.lengths)) != TRACEA_SUCCESS ||
      (st = read_rotation(op, positions, inv_freq, params.axes, params.sections, B, T, D, device, true, &r)) != TRACEA_SUCCESS)
    return st;
  const View *results[5] = {&c.k, &c.v, nullptr, nullptr, nullptr};
  int n = 2;
  if (c.e4m3) { results[n++] = &c.ks; results[n++] = &c.vs; }
  if (tq != nullptr) results[n++] = &qo;
  const View *reads[6] = {&k, &v, &starts, &c.table, nullptr, nullptr};
  int m = 4;
  if (tlengths != nullptr) reads[m++] = &lengths;
  if (tq != nullptr) reads[m++] = &q;
  for (int i = 0; i < n; ++i) {
    if (folds(*results[i])) return overlapping(op, "elements of a result share an address");
    if (over_rotation(r, *results[i])) return overlapping(op, "a result overlaps positions or inv_freq");
    for (int j = 0; j < m; ++j)
      if (!(results[i] == &qo && reads[j] == &q && same_view(qo, q)) && may_overlap(*results[i], *reads[j]))
        return overlapping(op, "a result overlaps an operand other than q_out its q, or that in part");
    for (int j = 0; j < i; ++j)
      if (may_overlap(*results[i], *results[j])) return overlapping(op, "results overlap each other");
  }
  if (B == 0 || T == 0 || (Hk == 0 && (tq == nullptr || q.shape[1] == 0))) return TRACEA_SUCCESS;
  a.k = head_view(k); a.v = head_view(v);
  a.Hk = (int)Hk;
  if (tq != nullptr) {
    a.q = head_view(q); a.q_out = head_view(qo);
    a.Hq = (int)q.shape[1];
  }
  a.kc = c.kp; a.vc = c.vp; a.ks = c.ksp; a.vs = c.vsp; a.table = c.pages;
  set_rotation(r, &a);
  a.B = (int)B; a.T = (int)T; a.D = (int)D;
  a.adjacent = params.adjacent != 0;
  for (a.vec = 8; a.vec > 1; a.vec /= 2) {
    bool fits = a.P % a.vec == 0;
    for (const View *t : operands) fits = fits && rows_on(*t, (size_t)(2 * a.vec));
    if (fits) break;
  }
  a.held = a.P % 4 == 0;
  for (const View *t : operands)
    a.held = a.held && rows_on(*t, 16) && t->stride[2] >= 0 && (t->stride[2] * std::min(T, (long long)c.pages.P) + D) * 2 < (1ll << 31);
  for (const View *t : {&c.k, &c.v}) a.held = a.held && (t->stride[2] * c.pages.P + D) * 2 < (1ll << 31);
  const long long pages = (T + c.pages.P - 2) / c.pages.P + 1;
  if (B > 65535 || pages >= (1 << 22) || T > (1ll << 31) - (1 << 16)) return fail(TRACEA_UNSUPPORTED_CONFIG, "%s: %lld sequences of %lld new tokens are more than is supported", op, B, T);
  a.pages = (int)pages;
  DeviceScope scope(device);
  if (scope.err != hipSuccess) return hip_status("hipSetDevice", (int)scope.err);
  // Workgroups for the heads of a page: a token's angles are worked out once for the heads of a workgroup, and a CU wants four with 64 tokens of
  // 128 columns, more of smaller ones.  Two prompts of 4096 tokens in pages of 64, workgroups for 8 / 4 / 2 heads: 61 / 52 / 52 us; of 16, for 8 /
  // 2: 111 / 50.
  const long long cus = (long long)device_limits().cus, heads = std::max(1ll, Hk), couples = std::min(T, (long long)c.pages.P) * ((D + 8) / 16);
  const long long smaller = couples <= 128 ? 4 : couples <= 256 ? 2 : 1;
  long long groups = std::min(heads, std::max((heads + kAppendHeads - 1) / kAppendHeads, 4 * smaller * cus / (B * pages)));
  a.heads = (int)((heads + groups - 1) / groups);
  groups = (heads + a.heads - 1) / a.heads;
  a.queries = (int)((a.Hq + groups - 1) / groups);
  if (pages * groups >= (1ll << 22)) return fail(TRACEA_UNSUPPORTED_CONFIG, "%s: %lld heads of %lld new tokens are more than is supported", op, Hk, T);
  a.groups = (int)groups;
  return hip_status("cache append launch", launch_cache_append(a, k.dtype, (hipStream_t)params.stream));
}

// ---- attention over a cache ---------------------------------------------------------------------------------------

TraceaStatus dispatch_attention_cached(const TraceaTensorView &tq, const TraceaTensorView &k_cache, const TraceaTensorView &v_cache,
                                       const TraceaTensorView *k_scale, const TraceaTensorView *v_scale,
                                       const TraceaTensorView &page_table, const TraceaTensorView *q_lengths,
                                       const TraceaTensorView &k_lengths, TraceaTensorView *to, TraceaTensorView *tlse,
                                       const TraceaAttentionParams &params) {
  const char *op = "tracea_attention_cached";
  TraceaStatus st;
  if ((st = ready(op)) != TRACEA_SUCCESS) return st;
  if (to == nullptr) return fail(TRACEA_INVALID_PARAMS, "%s: output view is NULL", op);
  View q, o, lse, ql, kl;
  AttentionCachedArgs a{};
  if ((st = read(op, "q", tq, 4, &q)) != TRACEA_SUCCESS || (st = read(op, "o", *to, 4, &o)) != TRACEA_SUCCESS ||
      (tlse != nullptr && (st = read(op, "lse", *tlse, 3, &lse)) != TRACEA_SUCCESS))
    return st;
  if (!is_half(q.dtype)) return fail(TRACEA_UNSUPPORTED_CONFIG, "%s: f16 or bf16 queries (got %s)", op, dtype_name(q.dtype));
  if (o.dtype != q.dtype) return fail(TRACEA_UNSUPPORTED_CONFIG, "%s: q and o must share one type", op);
  const long long B = q.shape[0], Hq = q.shape[1], Sq = q.shape[2], D = q.shape[3];
  if (!same_shape(q, o)) return fail(TRACEA_INVALID_PARAMS, "%s: q and o must be [B,Hq,Sq,D]", op);
  const int device = q.device;
  if ((st = check_device(op, device)) != TRACEA_SUCCESS) return st;
  if (o.device != device) return other_device(op);
  if (columns_apart(q) || columns_apart(o)) return fail(TRACEA_UNSUPPORTED_CONFIG, "%s: the head dimension must be contiguous", op);
  if (tlse != nullptr) {
    if (lse.dtype != TRACEA_DTYPE_FLOAT32 || lse.shape[0] != B || lse.shape[1] != Hq || lse.shape[2] != Sq)
      return fail(TRACEA_INVALID_PARAMS, "%s: lse must be f32 [B,Hq,Sq]", op);
    if (lse.device != device) return other_device(op);
  }
  if (D < 1 || D > 128) return fail(TRACEA_UNSUPPORTED_CONFIG, "%s: head dim %lld (multiples of 8 up to 128 supported)", op, D);
  Cache c;
  const long long Hk = k_cache.rank == 4 && k_cache.shape != nullptr ? (long long)k_cache.shape[1] : 0;
  if ((st = read_cache(op, k_cache, v_cache, k_scale, v_scale, page_table, q.dtype, device, B, Hk, D, &c)) != TRACEA_SUCCESS ||
      (st = read_counts(op, "q_lengths", q_lengths, B, device, &ql, &a.q_len)) != TRACEA_SUCCESS ||
      (st = read_counts(op, "k_lengths", &k_lengths, B, device, &kl, &a.k_len)) != TRACEA_SUCCESS)
    return st;
  const View *results[2] = {&o, tlse != nullptr ? &lse : nullptr};
  const View *reads[8] = {&q, &c.k, &c.v, &c.table, &kl, q_lengths != nullptr ? &ql : nullptr, c.e4m3 ? &c.ks : nullptr, c.e4m3 ? &c.vs : nullptr};
  for (const View *t : results) {
    if (t == nullptr) continue;
    if (folds(*t)) return overlapping(op, "elements of a result share an address");
    for (const View *s : reads)
      if (s != nullptr && may_overlap(*t, *s)) return overlapping(op, "a result overlaps an operand");
  }
  if (tlse != nullptr && may_overlap(o, lse)) return overlapping(op, "results overlap each other");
  if (B == 0 || Hq == 0 || Sq == 0) return TRACEA_SUCCESS;
  if (Hk == 0 || Hq % Hk != 0)
    return fail(TRACEA_INVALID_PARAMS, "%s: %lld query heads are not a multiple of %lld key/value heads", op, Hq, Hk);
  const long long G = Hq / Hk;
  // (rows are divided by G with a 32-bit product)
  if (G * G * (Sq + 128) >= (1ll << 31))
    return fail(TRACEA_UNSUPPORTED_CONFIG, "%s: %lld queries of %lld heads a key/value head are more than is supported", op, Sq, G);
  float scale = params.scale;
  if (scale == 0.0f) scale = 1.0f / sqrtf((float)D);
  if (!std::isfinite(scale)) return fail(TRACEA_INVALID_PARAMS, "%s: scale is not finite", op);
  a.q = head_view(q); a.o = head_view(o);
  if (tlse != nullptr) {
    a.lse = (float *)lse.ptr;
    a.lse_sb = lse.stride[0]; a.lse_sh = lse.stride[1]; a.lse_ss = lse.stride[2];
  }
  a.k = c.kp; a.v = c.vp; a.ks = c.ksp; a.vs = c.vsp; a.table = c.pages;
  if (c.pages.N == 0) a.table.M = 0;
  const long long per_page = c.pages.P / 16;
  a.page_magic = per_page > 1 ? (unsigned)(((1ull << 32) + per_page - 1) / per_page) : 0;
  a.B = (int)B; a.Hk = (int)Hk; a.G = (int)G; a.Sq = (int)Sq; a.D = (int)D;
  a.g_magic = G > 1 ? (unsigned)(((1ull << 32) + G - 1) / G) : 0;
  a.negate = scale < 0.0f;
  a.scale_log2 = fabsf(scale) * 1.4426950408889634f;
  a.causal = params.causal ? 1 : 0;
  a.q_vec = rows_on(q, 16);
  a.o_vec = rows_on(o, 16);
  const long long rows = G * Sq;
  // Blocks of 128 rows share tiles of keys through LDS, blocks of 16 or 32 read them straight into registers.
  a.rows = rows > 64 ? 128 : rows > 16 ? 32 : 16;
  const bool tiles = a.rows == 128;
  a.step = tiles ? kCachedTile : kCachedStep;
  a.step_log2 = tiles ? 6 : 7;
  a.row_blocks = (int)((rows + a.rows - 1) / a.rows);
  a.splits = 1;
  const long long problems = B * Hk * a.row_blocks;
  if (problems >= (1ll << 24)) return fail(TRACEA_UNSUPPORTED_CONFIG, "%s: more workgroups than a launch can have", op);
  DeviceScope scope(device);
  if (scope.err != hipSuccess) return hip_status("hipSetDevice", (int)scope.err);
  hipStream_t stream = (hipStream_t)params.stream;
  std::lock_guard<std::mutex> together(g_launches);
  const long long cus = (long long)device_limits().cus, most = std::max(1ll, ((long long)a.table.M * c.pages.P + a.step - 1) / a.step);
  const double width_of = D <= 64 ? 0.5 : 1.0;
  long long slots = 0;
  a.slots = tiles ? 1 : 2;
  if (tiles) {
    a.splits = plan_tiles(problems, most, c.e4m3, width_of, cus);
    slots = a.splits > 1 ? problems * a.splits : 0;
  } else if (shares_pay(problems, most, c.e4m3, width_of, a.rows)) {
    // Every problem by itself, where shares are of few steps and their parts fill the device about evenly: in a line many workgroups
    // would have the end of one problem and the beginning of the next, which costs more than a step.  Parts for one workgroup a CU (two of 64
    // columns), or for two where there are problems enough to keep the join short.  us in a line / by themselves: B16, 20 rows, 2000 keys of 96
    // columns (parts of 3 steps) 20.3 / 18.4; B2 20000 (5) 22.9 / 20.1; one query, D128, B8 4096 keys (two of 3 steps a CU) 19.2 / 17.3 in 8 bits, 26.0 /
    // 21.0 in 16.  In parts of 6 and more what is uneven costs more: B8 8192 keys of 16 bits 40 / 46.
    // In a line, two workgroups a CU where most have more than one problem: B32 4096 keys of 8 bits 51.8 / 45.8 us; else one, which leaves half
    // the parts: B8 8192 26.5 / 25.7, of 16 bits 41.5 / 40.5.
    a.shares = (int)(D <= 64 ? 2 * cus : cus);
    a.line = (int)(D <= 64 || 2 * problems > cus ? 2 * cus : cus);
    a.workgroups = a.line;
    if (problems <= a.shares) {
      a.apart = 5;
      a.twice = D > 64 && 8 * problems >= cus ? 3 : a.apart;
      a.workgroups = 2 * a.shares;
    }
    slots = 2 * a.workgroups;
  }
  a.all_slots = (int)slots;
  if (slots > 0) {
    const size_t n = (size_t)(slots * a.rows), width = D <= 64 ? 64 : 128;
    a.part_o = (float *)train_scratch(device, stream, n * (width + 2) * 4 + (size_t)problems * 8);
    if (a.part_o != nullptr) {
      a.part_ml = a.part_o + n * width;
      a.meta = (int *)(a.part_ml + 2 * n);
    } else {  // (slower, the same result to rounding)
      a.workgroups = 0;
      a.splits = 1;
    }
  }
  return hip_status("attention over a cache launch", launch_attention_cached(a, q.dtype, c.e4m3, stream));
}

}  // namespace tracea_amd
