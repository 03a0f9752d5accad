// Attention for training, gfx950: a forward pass that keeps each row's log-sum-exp and a backward pass that recomputes the
// probabilities from it.
//
//   s_ij = scale q_i . k_j  over the keys a row sees (j < its sequence's key length; causal: j <= i + keys - queries)
//   lse_i = log sum_j exp(s_ij)      o_i = sum_j exp(s_ij - lse_i) v_j        (no key: lse -inf, o 0)
//   P_ij = exp(s_ij - lse_i)   delta_i = dO_i . O_i   dS_ij = P_ij (dO_i . v_j - delta_i)
//   dV_j = sum_i P_ij dO_i     dK_j = scale sum_i dS_ij q_i     dQ_i = scale sum_j dS_ij k_j
// P and dS are rounded to the operand type for the second products, and delta comes from O as the forward pass rounded it: the price of
// products at the 16-bit rate and of one pass for delta.  Errors in 2-norm are 1.3 to 1.57 times those of 32-bit arithmetic rounded
// once, most for dQ and dK of rows with few keys, where the rounding of O averages out least.
//
// Three walks of one shape.  A wave owns 32 columns whose operand fragments stay in registers and streams the other
// side in tiles of 64 through LDS (32: with D = 128 the sums of dK and dV are half of the 256 registers that leave room for two
// waves on a SIMD, and the products of one fill the gaps of the other); every product is v_mfma_f32_16x16x32 with fp32 sums.  In the result of a 16x16 block
// lane l holds column l & 15 and rows 4 (l >> 4) + 0..3; two blocks one above the other, converted to 16 bits, are the
// second operand of the next product over those 32 rows (k slots 0-3: rows 4 g + e, slots 4-7: rows 16 + 4 g + e,
// g = l >> 4), whose first operand enumerates the same rows: two transposing reads of the tile.
//   forward  columns = query rows, stream K and V:    S^T = K Q^T, O^T += V^T P^T
//   dQ       columns = query rows, stream K and V:    S^T, dP^T = V dO^T, dQ^T += K^T dS^T
//   dK, dV   columns = keys, stream Q and dO:         S = Q K^T, dP = dO V^T, dV^T += dO^T P, dK^T += Q^T dS
// dQ has a walk of its own although that computes S and dP twice (7 products instead of 5): sums over the keys of a
// row would otherwise meet from different workgroups, in an order that changes from run to run.  Both walks are one launch.
//
// The rows of a head that shares its keys with G - 1 others are packed, r = query G + head of the group: a tile of K and V is read
// once for all of them, and the sums over the heads of a group in dK and dV are sums over rows.
#include <type_traits>

#include "attention_tile.hpp"
#include "train.hpp"

namespace tracea_amd {

namespace {

// Probabilities and their gradients become 16-bit operands.  f16 has no range for either: a row over thousands of keys has
// probabilities below its smallest normal number.  Backward, P is kept as 2^14 P, dS scaled by a power of two from the largest
// |dP - delta| there can be (see ds_scale); forward, see P_SHIFT.  All factors leave with the results.  bf16 needs none.
constexpr float F16_P_SHIFT = 14.0f;

template <int DT>
__device__ __forceinline__ void unpack8(u32x4 w, float (&x)[8]) {
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if constexpr (DT == DT_F16) {
      x[2 * e] = (float)__builtin_bit_cast(_Float16, (unsigned short)(w[e] & 0xffffu));
      x[2 * e + 1] = (float)__builtin_bit_cast(_Float16, (unsigned short)(w[e] >> 16));
    } else {
      x[2 * e] = __builtin_bit_cast(float, w[e] << 16);
      x[2 * e + 1] = __builtin_bit_cast(float, w[e] & 0xffff0000u);
    }
  }
}

__device__ __forceinline__ void dma4(u32x4 rsrc, unsigned offset, unsigned lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dword %1, %2, 0 offen lds" ::"s"(lds), "v"(offset), "s"(rsrc) : "memory");
}
// The block and the (batch, key/value head) of workgroup `id` of blocks * B * Hk, blocks numbered from the one with most work.
// Dense: an XCD has a run of them.  Causal: the heaviest blocks of all heads first; a head stays on one XCD where their number is a
// multiple of 8.  With lengths a head's blocks go round the XCDs, which otherwise would get sequences of unequal lengths.
struct Slot {
  int blk, bh;
};
__device__ __forceinline__ Slot slot_of(const AttentionTrainArgs &a, int id, int blocks) {
  const int heads = a.B * a.Hk;
  if (a.order == 0) {
    const int vid = xcd_run(id, heads * blocks), bh = vid / blocks;
    return {vid - bh * blocks, bh};
  }
  const int blk = id / heads, bh = id - blk * heads;
  return {blk, a.order == 1 ? bh : (bh + blk) % heads};
}

struct Rows {  // of one batch entry and key/value head
  int b, hk, lq, lk, off;  // lengths; a causal row of query i sees keys up to i + off
};
__device__ __forceinline__ Rows rows_of(const AttentionTrainArgs &a, int bh) {
  Rows r;
  r.b = bh / a.Hk;
  r.hk = bh - r.b * a.Hk;
  r.lq = a.Sq;
  r.lk = a.Sk;
  if (a.q_len != nullptr) r.lq = min(max(a.q_len[r.b], 0), a.Sq);
  if (a.k_len != nullptr) r.lk = min(max(a.k_len[r.b], 0), a.Sk);
  r.off = r.lk - r.lq;
  return r;
}
__device__ __forceinline__ int query_of(const AttentionTrainArgs &a, int r) {
  return a.G == 1 ? r : (int)__umulhi((unsigned)r, a.g_magic);
}
__device__ __forceinline__ long long row_at(const AttentionTrainArgs &a, const HeadView &t, const Rows &w, int r) {
  const int i = query_of(a, r);
  return (long long)w.b * t.sb + (long long)(w.hk * a.G + (r - i * a.G)) * t.sh + (long long)i * t.ss;
}
__device__ __forceinline__ const unsigned short *slice(const HeadView &t, int b, int h) {
  return (const unsigned short *)t.p + (long long)b * t.sb + (long long)h * t.sh;
}

// Fragment of 16 resident rows for the k-step ks: lane l holds row l & 15, columns 32 ks + 8 (l >> 4) .. + 7.
__device__ __forceinline__ u32x4 resident(const unsigned short *row, bool there, int col, int D) {
  u32x4 z = {0, 0, 0, 0};
  return there && col < D ? *(const u32x4 *)(row + col) : z;
}

// Adds the accumulators of the second of two waves that share columns to the first's, through LDS (the tiles are done with).
template <int N, typename F>
__device__ __forceinline__ void join_halves(unsigned char *lds, int group, int half, int lane, F &&acc) {
  f32x4 *at = (f32x4 *)lds + group * N * 64 + lane;
  __syncthreads();
  if (half == 1) {
#pragma unroll
    for (int i = 0; i < N; ++i) at[i * 64] = acc(i);
  }
  __syncthreads();
  if (half == 0) {
#pragma unroll
    for (int i = 0; i < N; ++i) acc(i) += at[i * 64];
  }
}

// The power of two that dS is multiplied by before it becomes an f16 operand: |dP - delta| <= 2 max|dO| max|V|
// (delta is a mean of the dP of its row), and P <= 1.
__device__ __forceinline__ float ds_scale(const AttentionTrainArgs &a, int bh, int lane) {
  const float *n = a.norms + (long long)bh * a.norm_blocks;
  const int of_rows = a.rows_pad / TILE;
  float mo = 0.0f, mv = 0.0f;
  for (int i = lane; i < a.norm_blocks; i += 64) {
    const float x = n[i];
    if (i < of_rows) mo = fmaxf(mo, x);
    else mv = fmaxf(mv, x);
  }
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) {
    mo = fmaxf(mo, __shfl_xor(mo, m, 64));
    mv = fmaxf(mv, __shfl_xor(mv, m, 64));
  }
  const float bound = 2.0f * sqrtf(mo) * sqrtf(mv);
  int e = 14;
  if (bound > 0.0f && bound < 3.0e38f) (void)frexpf(bound, &e);  // bound < 2^e
  e = 14 - e;
  e = e < -100 ? -100 : e > 100 ? 100 : e;
  return __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane((127 + e) << 23));
}

// ---- forward --------------------------------------------------------------------------------------------------

// Forward: one pass over the keys with a running reference and sum per row.  A wave's scores of tile t + 1 are computed under the
// exponentials of tile t, and P V of tile t under the maximum over t + 1, so that K is a tile ahead of V.  SG = 2: two waves share
// their rows and walk every other tile of 64 keys; their states are joined at the end.  A wave has 16 NQ rows: 32, or 16 for a token
// or two of some heads, where the empty half would be most of what it waits for.
// Bound, long rows: vector work (exponential, maximum and conversion of a score cost about as many cycles as its products do) beside
// the matrix pipe, and power: B4 H32 S4096 bf16 D128 1030-1100 us by card = 1.00-1.07 PFLOP/s, f16 D64 697-722 us = 0.76-0.79.  One query over a long
// cache: reading K and V, B8 H32:8 D128 over 8192 keys 47 us = 5.7 TB/s with the join (a large copy reaches 4.8; part of it is in the
// memory-side cache).  (Two waves a SIMD are what the registers are limited for; the tiles of SG = 2 at D above 64, 128 KB, leave room
// for one workgroup, and so for one wave.)
template <int DT, int DL, int DU, int WAVES, int SG, int NQ>
__global__ void __launch_bounds__(WAVES * 64) __attribute__((amdgpu_waves_per_eu(2, 2)))
attention_train_forward_kernel(const AttentionTrainArgs a) {
  using T = Tile<DL>;
  constexpr int WR = 16 * NQ, BR = WR * WAVES / SG, KS = DU / 32, DB = DU / 16, KB = TILE / 16, STEP = SG * TILE;  // keys of a step
  constexpr unsigned SIDE = SG * T::BYTES, V_AT = 2 * SIDE;  // two steps of K, two of V
  __shared__ __attribute__((aligned(1024))) unsigned char sK[4 * SIDE];

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r16 = lane & 15, g4 = lane >> 4, group = wave / SG, kg = wave % SG;
  const int blocks = (a.G * a.Sq + BR - 1) / BR;
  const Slot slot = slot_of(a, blockIdx.x, blocks);
  const int bh = slot.bh, blk = blocks - 1 - slot.blk;  // most keys under a causal mask first
  const Rows w = rows_of(a, bh);
  const int rows = a.G * w.lq;
  const int r_wave = blk * BR + group * WR;

  const int last_row = min(blk * BR + BR, rows) - 1;
  int keys = 0;  // that any row of the block sees
  if (last_row >= blk * BR) keys = a.causal ? min(w.lk, query_of(a, last_row) + w.off + 1) : w.lk;
  int steps = keys > 0 ? (keys + STEP - 1) / STEP : 0, s0 = 0;
  if (a.splits > 1) {
    s0 = (int)blockIdx.y * a.steps_per_split;
    steps = min(steps, s0 + a.steps_per_split);
  }

  const unsigned short *Kg = slice(a.k, w.b, w.hk), *Vg = slice(a.v, w.b, w.hk);
  auto request = [&](const unsigned short *base, long long ss, int step, unsigned side) __attribute__((always_inline)) {
    const int lane_ = fresh(lane);
    const unsigned bytes = (unsigned)ss * 2u;
#pragma unroll
    for (int g = 0; g < SG; ++g) {
      const int tile = step * SG + g, left = w.lk - tile * TILE;
      const unsigned char *dst = sK + side + (unsigned)(step & 1) * SIDE + g * T::BYTES;
      const unsigned short *at = base + (long long)tile * TILE * ss;
      constexpr int APART = WAVES * 64 / T::CH;
      if (left >= TILE) load_tile<DL, WAVES>(at, (long long)bytes * APART, dst, a.D, lane_, wave, [&](int row) { return row * bytes; });
      else load_tile_any<DL, WAVES>(at, dst, a.D, lane_, wave, [&](int row) { return row < left ? row * bytes : BEYOND; });
    }
  };
  auto request_k = [&](int step) __attribute__((always_inline)) { request(Kg, a.k.ss, step, 0); };
  auto request_v = [&](int step) __attribute__((always_inline)) { request(Vg, a.v.ss, step, V_AT); };
  if (s0 < steps) {  // (in flight while the rest is set up)
    request_k(s0);
    request_v(s0);
    if (s0 + 1 < steps) request_k(s0 + 1);
  }

  int q_last[NQ];  // the last key that the lane's queries see
  u32x4 qf[NQ][KS];
#pragma unroll
  for (int qb = 0; qb < NQ; ++qb) {
    const int r = r_wave + qb * 16 + r16;
    const bool there = r < rows;
    q_last[qb] = !there ? -1 : a.causal ? min(w.lk - 1, query_of(a, r) + w.off) : w.lk - 1;
    const unsigned short *p = (const unsigned short *)a.q.p + (there ? row_at(a, a.q, w, r) : 0);
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      qf[qb][ks] = resident(p, there, ks * 32 + g4 * 8, a.D);
      if (a.negate) qf[qb][ks] ^= 0x80008000u;
    }
  }
  // of the wave: keys that some row sees, and the first that not every row sees; as steps: those with a tile of its own that some row
  // sees, and those whose tile every row sees whole
  int wave_keys = 0, wave_full = 0;
  if (r_wave < rows) {
    const int r_end = min(r_wave + WR, rows) - 1;
    wave_keys = a.causal ? min(w.lk, query_of(a, r_end) + w.off + 1) : w.lk;
    wave_full = a.causal ? min(w.lk, query_of(a, r_wave) + w.off + 1) : w.lk;  // (what rows past the end hold is dropped)
  }
  const int wave_steps = wave_keys > kg * TILE ? min(steps, (wave_keys - kg * TILE + STEP - 1) / STEP) : 0;
  const int full_steps = wave_full >= (kg + 1) * TILE ? min(wave_steps, (wave_full - kg * TILE) / TILE / SG + ((wave_full - kg * TILE) / TILE % SG != 0)) : 0;


  f32x4 o[NQ][DB];
  // reference (log2 units) and sum of the lane's keys.  The sum has 64 bits: a tile behind thousands of others, or in a row with one
  // large probability, adds a small number to a large one (in 32 bits lse was off by 1e-4 over 131072 keys; dense calls take the same
  // time either way, S1024 D64 causal 15.2 us, with 32 bits 14.9)
  float m[NQ];
  double total[NQ];
#pragma unroll
  for (int qb = 0; qb < NQ; ++qb) {
    m[qb] = -INFINITY;
    total[qb] = 0.0;
#pragma unroll
    for (int d = 0; d < DB; ++d) o[qb][d] = f32x4{0, 0, 0, 0};
  }

  const unsigned rows0 = rows_base<DL>(sK, r16, g4) + kg * T::BYTES, cols0 = columns_base<DL>(sK, r16, g4) + kg * T::BYTES;
  // What a row does not see becomes -inf; the largest score of the lane's in tile `step`, one value at a time.
  auto take_max = [&](int step, int v, f32x4 (&z)[NQ][KB], float (&mx)[NQ], auto edge_tag) __attribute__((always_inline)) {
    const int qb = v >> 4, kb = (v >> 2) & 3, e = v & 3;
    if constexpr (decltype(edge_tag)::value)
      z[qb][kb][e] = (step * SG + kg) * TILE + kb * 16 + g4 * 4 + e > q_last[qb] ? -INFINITY : z[qb][kb][e];
    mx[qb] = fmaxf(mx[qb], z[qb][kb][e]);
  };
  // The rows' references, and what is summed up already, where a tile exceeds the scores they stand for by LAZY_MAX powers of two.
  auto move_reference = [&](const float (&mx)[NQ]) __attribute__((always_inline)) {
    bool moved = false;
    float alpha[NQ];
#pragma unroll
    for (int qb = 0; qb < NQ; ++qb) {
      const float top = groups_max_valu(mx[qb]) * a.scale_log2;
      const bool mv = top > m[qb] + (P_SHIFT<DT> + LAZY_MAX<DT>);  // (a first score above -inf always moves it)
      const float mn = mv ? top - P_SHIFT<DT> : m[qb];
      alpha[qb] = mv ? __builtin_amdgcn_exp2f(m[qb] - mn) : 1.0f;
      m[qb] = mn;
      moved |= mv;
    }
    if (__any(moved)) {
#pragma unroll
      for (int qb = 0; qb < NQ; ++qb) {
        total[qb] *= (double)alpha[qb];
#pragma unroll
        for (int d = 0; d < DB; ++d) o[qb][d] *= alpha[qb];
      }
    }
  };

  // One step: P of the scores `z` of step t, its P V, and, unless LAST, the scores `zn` of step t + 1 (EDGE: masked) and their maximum.
  // One chunk per first-operand fragment, read AHEAD chunks before.
  constexpr int AHEAD = 2;
  auto iterate = [&](int t, f32x4 (&z)[NQ][KB], f32x4 (&zn)[NQ][KB], auto edge_tag, auto last_tag) __attribute__((always_inline)) {
    constexpr bool LAST = decltype(last_tag)::value;
    constexpr int N1 = LAST ? 0 : KB * KS, N2 = 2 * DB, N = N1 + N2;
    const unsigned at_k = fresh(rows0) + (unsigned)((t + 1) & 1) * SIDE, at_v = fresh(cols0) + (unsigned)(t & 1) * SIDE;
    u32x4 frag[AHEAD + 1], pf[NQ][2];
    float mx[NQ], ref[NQ], sum[NQ];
#pragma unroll
    for (int qb = 0; qb < NQ; ++qb) {
      mx[qb] = -INFINITY;
      ref[qb] = m[qb] == -INFINITY ? 0.0f : m[qb];  // (nothing visible yet: exp2(-inf) = 0)
      sum[qb] = 0.0f;
    }
    auto read = [&](auto tag) __attribute__((always_inline)) {
      constexpr int i = decltype(tag)::value;
      if constexpr (i < N1) frag[i % (AHEAD + 1)] = read_rows<DL>(at_k, 0, i % KB, i / KB);
      else if constexpr (i < N) frag[i % (AHEAD + 1)] = read_columns<DL>(at_v, V_AT, (i - N1) / DB, (i - N1) % DB);
    };
    auto probability = [&](int v) __attribute__((always_inline)) {
      const int qb = v >> 4, kb = (v >> 2) & 3, e = v & 3;
      const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(z[qb][kb][e], a.scale_log2, -ref[qb]));
      sum[qb] += p;
      z[qb][kb][e] = p;
      if ((v & 7) == 7) pf[qb][kb >> 1] = pack_operand<DT>(z[qb][kb - 1], z[qb][kb]);
    };
    static_for<0, AHEAD>([&](auto tag) __attribute__((always_inline)) { read(tag); });
    if constexpr (LAST) {
#pragma unroll
      for (int v = 0; v < 16 * NQ; ++v) probability(v);
    }
    static_for<0, N>([&](auto tag) __attribute__((always_inline)) {
      constexpr int i = decltype(tag)::value;
      const u32x4 &f = frag[i % (AHEAD + 1)];
      read(std::integral_constant<int, i + AHEAD>{});
      if constexpr (i < N1) {
        constexpr int kb = i % KB, ks = i / KB, PER = (16 * NQ + N1 - 1) / (LAST ? 1 : N1);
#pragma unroll
        for (int qb = 0; qb < NQ; ++qb) zn[qb][kb] = Mfma16<DT>::run(f, qf[qb][ks], ks == 0 ? f32x4{0, 0, 0, 0} : zn[qb][kb]);
#pragma unroll
        for (int v = i * PER; v < (i + 1) * PER && v < 16 * NQ; ++v) probability(v);
      } else {
        constexpr int j = i - N1, s = j / DB, d = j % DB, PER = (16 * NQ + N2 - 1) / N2;
#pragma unroll
        for (int qb = 0; qb < NQ; ++qb) o[qb][d] = Mfma16<DT>::run(f, pf[qb][s], o[qb][d]);
        if constexpr (!LAST) {
#pragma unroll
          for (int v = j * PER; v < (j + 1) * PER && v < 16 * NQ; ++v) take_max(t + 1, v, zn, mx, edge_tag);
        }
      }
      fence();
    });
#pragma unroll
    for (int qb = 0; qb < NQ; ++qb) total[qb] += (double)sum[qb];
    if constexpr (!LAST) move_reference(mx);
  };
  // Step t: the scores of t are there; K of t + 1 and V of t have arrived, K of t + 2 and V of t + 1 go out.
  auto head = [&](int t) __attribute__((always_inline)) {
    __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0)
    __syncthreads();
    if (t + 2 < steps) request_k(t + 2);
    if (t + 1 < steps) request_v(t + 1);
  };

  f32x4 za[NQ][KB], zb[NQ][KB];
  int t = s0;
  if (t < steps) {
    __builtin_amdgcn_s_waitcnt(0x0f70);
    __syncthreads();
    if (t < wave_steps) {  // the first scores, on their own
      const unsigned at_k = fresh(rows0) + (unsigned)(t & 1) * SIDE;
      float mx[NQ];
#pragma unroll
      for (int qb = 0; qb < NQ; ++qb) mx[qb] = -INFINITY;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) {
          const u32x4 kf = read_rows<DL>(at_k, 0, kb, ks);
#pragma unroll
          for (int qb = 0; qb < NQ; ++qb) za[qb][kb] = Mfma16<DT>::run(kf, qf[qb][ks], ks == 0 ? f32x4{0, 0, 0, 0} : za[qb][kb]);
        }
#pragma unroll
      for (int v = 0; v < 16 * NQ; ++v) take_max(t, v, za, mx, std::true_type{});
      move_reference(mx);
    }
  }
  const int whole = full_steps - 1, last = wave_steps - 1;  // steps whose next one is whole; the wave's last
  auto back = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int qb = 0; qb < NQ; ++qb)
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) za[qb][kb] = zb[qb][kb];
  };
  for (; t + 1 < whole; t += 2) {
    head(t);
    iterate(t, za, zb, std::false_type{}, std::false_type{});
    head(t + 1);
    iterate(t + 1, zb, za, std::false_type{}, std::false_type{});
  }
  for (; t < last; ++t) {
    head(t);
    iterate(t, za, zb, std::true_type{}, std::false_type{});
    back();
  }
  if (t == last && t >= s0) {
    head(t);
    iterate(t, za, zb, std::true_type{}, std::true_type{});
    ++t;
  }
  for (; t < steps; ++t) head(t);  // (tiles that only other waves see)
  float l[NQ];
#pragma unroll
  for (int qb = 0; qb < NQ; ++qb) l[qb] = (float)total[qb];

  if constexpr (SG == 2) {  // the second wave's state to the first
    f32x4 *const at = (f32x4 *)sK + group * (NQ * DB + 1) * 64 + lane;
    __syncthreads();
    if (kg == 1) {
#pragma unroll
      for (int i = 0; i < NQ * DB; ++i) at[i * 64] = o[i / DB][i % DB];
      at[NQ * DB * 64] = f32x4{m[0], m[NQ - 1], l[0], l[NQ - 1]};
    }
    __syncthreads();
    if (kg == 1) return;
    const f32x4 ml = at[NQ * DB * 64];
#pragma unroll
    for (int qb = 0; qb < NQ; ++qb) {
      const float top = fmaxf(m[qb], ml[qb]), ref = top == -INFINITY ? 0.0f : top;
      const float f0 = __builtin_amdgcn_exp2f(m[qb] - ref), f1 = __builtin_amdgcn_exp2f(ml[qb] - ref);
      m[qb] = top;
      l[qb] = f0 * l[qb] + f1 * ml[2 + qb];
#pragma unroll
      for (int d = 0; d < DB; ++d) o[qb][d] = f0 * o[qb][d] + f1 * at[(qb * DB + d) * 64];
    }
  }

#pragma unroll
  for (int qb = 0; qb < NQ; ++qb) {
    const int r = r_wave + qb * 16 + r16;
    float sum = groups_sum(l[qb]);
    if (r >= a.G * a.Sq) continue;
    if (r >= rows) {  // a query behind its sequence's length
      m[qb] = -INFINITY;
      sum = 0.0f;
#pragma unroll
      for (int d = 0; d < DB; ++d) o[qb][d] = f32x4{0, 0, 0, 0};
    }
    if (a.splits > 1) {
      const long long at = ((long long)blockIdx.y * a.B * a.Hk + bh) * ((long long)a.G * a.Sq) + r;
      if (g4 == 0) {
        a.part_ml[2 * at] = m[qb];
        a.part_ml[2 * at + 1] = sum;
      }
#pragma unroll
      for (int d = 0; d < DB; ++d)
        if (d * 16 + g4 * 4 < a.D) *(f32x4 *)(a.part_o + at * DU + d * 16 + g4 * 4) = o[qb][d];
      continue;
    }
    const float inv = sum > 0.0f ? 1.0f / sum : sum == 0.0f ? 0.0f : sum;  // (NaN stays)
    unsigned short *p = (unsigned short *)a.o.p + row_at(a, a.o, w, r);
#pragma unroll
    for (int d = 0; d < DB; ++d)
      if (d * 16 + g4 * 4 < a.D) *(u32x2 *)(p + d * 16 + g4 * 4) = pack_result<DT>(o[qb][d], inv);
    if (g4 == 0) {
      const int i = query_of(a, r);
      a.lse[(long long)w.b * a.lse_sb + (long long)(w.hk * a.G + r - i * a.G) * a.lse_sh + (long long)i * a.lse_ss] =
          sum == 0.0f ? -INFINITY : (m[qb] + __builtin_amdgcn_logf(sum)) * LN2;
    }
  }
}

// Joins the partial results of a split key axis: a row per 32 lanes, which load one part's reference and sum each (at most 32
// parts) and 4 columns of every part's o.  Bound by the latency of its loads: 4 to 5 us for 256 rows of 8 parts.
template <int DT, int DU>
__global__ void __launch_bounds__(256) attention_train_join_kernel(const AttentionTrainArgs a) {
  const long long id = ((long long)blockIdx.x * 256 + threadIdx.x) / 32;
  const int lane = threadIdx.x & 31, c = lane * 4, per = a.G * a.Sq;
  if (id >= (long long)a.B * a.Hk * per) return;
  const int bh = (int)(id / per), r = (int)(id - (long long)bh * per);
  const Rows w = rows_of(a, bh);
  const long long plane = (long long)a.B * a.Hk * per, at = (long long)bh * per + r;
  const float own_m = lane < a.splits ? a.part_ml[2 * (lane * plane + at)] : -INFINITY;
  const float own_l = lane < a.splits ? a.part_ml[2 * (lane * plane + at) + 1] : 0.0f;
  float m = own_m;
#pragma unroll
  for (int s = 1; s < 32; s <<= 1) m = fmaxf(m, __shfl_xor(m, s, 32));
  const float own_f = __builtin_amdgcn_exp2f(own_m - (m == -INFINITY ? 0.0f : m));
  float sum = own_f * own_l;
#pragma unroll
  for (int s = 1; s < 32; s <<= 1) sum += __shfl_xor(sum, s, 32);
  f32x4 o = {0, 0, 0, 0};
  const float *from = a.part_o + at * DU + (c < a.D ? c : 0);
#pragma unroll 8
  for (int s = 0; s < a.splits; ++s) o += __shfl(own_f, s, 32) * *(const f32x4 *)(from + s * plane * DU);
  const float inv = sum > 0.0f ? 1.0f / sum : sum == 0.0f ? 0.0f : sum;
  if (c < a.D) *(u32x2 *)((unsigned short *)a.o.p + row_at(a, a.o, w, r) + c) = pack_result<DT>(o, inv);
  if (c == 0) {
    const int i = query_of(a, r);
    a.lse[(long long)w.b * a.lse_sb + (long long)(w.hk * a.G + r - i * a.G) * a.lse_sh + (long long)i * a.lse_ss] =
        sum == 0.0f ? -INFINITY : (m + __builtin_amdgcn_logf(sum)) * LN2;
  }
}

// ---- backward ---------------------------------------------------------------------------------------------------

// Per packed row -lse log2(e) and -(dO . O), which both walks need; f16: the largest squared norms of 64 rows of dO, and of 64 keys of V.
// Bound by reading dO and O: B4 H32 S4096 D128 bf16 48.5 us = 5.5 TB/s; a launch's 5 us at B1 H12 S197 D64.
template <int DT>
__global__ void __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(4))) attention_train_rows_kernel(const AttentionTrainArgs a) {
  constexpr int LPR = 16;  // lanes per row, 8 columns each
  __shared__ float s_max[4];
  const int c = (threadIdx.x % LPR) * 8, row_blocks = a.rows_pad / TILE, blocks = DT == DT_F16 ? a.norm_blocks : row_blocks;
  const int bh = (int)blockIdx.x / blocks, blk = (int)blockIdx.x - bh * blocks;
  const Rows w = rows_of(a, bh);
  const bool of_rows = blk < row_blocks;
  // (all loads first: a launch of few blocks is as long as the waits one after another)
  u32x4 xs[TILE / 16], ys[TILE / 16];
  float lse[TILE / 16];
#pragma unroll
  for (int it = 0; it < TILE / 16; ++it) {
    const int row = it * 16 + (int)threadIdx.x / LPR, r = blk * TILE + row, j = r - row_blocks * TILE;
    xs[it] = ys[it] = u32x4{0, 0, 0, 0};
    lse[it] = -INFINITY;
    if (of_rows && r < a.G * w.lq) {
      if (c < a.D) {
        xs[it] = *(const u32x4 *)((const unsigned short *)a.d_o.p + row_at(a, a.d_o, w, r) + c);
        ys[it] = *(const u32x4 *)((const unsigned short *)a.o.p + row_at(a, a.o, w, r) + c);
      }
      const int i = query_of(a, r);
      lse[it] = a.lse[(long long)w.b * a.lse_sb + (long long)(w.hk * a.G + r - i * a.G) * a.lse_sh + (long long)i * a.lse_ss];
    } else if (!of_rows && j < w.lk && c < a.D) {
      xs[it] = *(const u32x4 *)(slice(a.v, w.b, w.hk) + (long long)j * a.v.ss + c);
    }
  }
  float big = 0.0f;
#pragma unroll
  for (int it = 0; it < TILE / 16; ++it) {
    const int r = blk * TILE + it * 16 + (int)threadIdx.x / LPR;
    float x[8], y[8], dot = 0.0f, norm = 0.0f;
    unpack8<DT>(xs[it], x);
    unpack8<DT>(ys[it], y);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      dot = __builtin_fmaf(x[e], y[e], dot);
      norm = __builtin_fmaf(x[e], x[e], norm);
    }
    if (of_rows) {
#pragma unroll
      for (int s = 1; s < LPR; s <<= 1) dot += __shfl_xor(dot, s, 64);
      if (c == 0) {
        const bool sees = lse[it] != -INFINITY;
        a.neg_lse2[(long long)bh * a.rows_pad + r] = sees ? (DT == DT_F16 ? F16_P_SHIFT : 0.0f) - lse[it] * LOG2E : -INFINITY;
        a.neg_delta[(long long)bh * a.rows_pad + r] = sees ? -dot : 0.0f;
      }
    }
    if constexpr (DT == DT_F16) {
#pragma unroll
      for (int s = 1; s < LPR; s <<= 1) norm += __shfl_xor(norm, s, 64);
      big = fmaxf(big, norm);
    }
  }
  if constexpr (DT == DT_F16) {
    big = groups_max(big);
    if ((threadIdx.x & 63) == 0) s_max[threadIdx.x >> 6] = big;
    __syncthreads();
    if (threadIdx.x == 0) a.norms[(long long)bh * a.norm_blocks + blk] = fmaxf(fmaxf(s_max[0], s_max[1]), fmaxf(s_max[2], s_max[3]));
  }
}

// dQ of a block of packed rows: three products and two operands from LDS per tile.  SG = 2: two waves share 32 rows, each takes half of
// every tile of keys.
template <int DT, int DL, int DU, int WAVES, int SG>
__device__ __forceinline__ void dq_block(const AttentionTrainArgs &a, int id, unsigned char *sK) {
  using T = Tile<DL>;
  constexpr int BR = 32 * WAVES / SG, KS = DU / 32, DB = DU / 16;
  constexpr unsigned V_AT = 2 * T::BYTES;  // two tiles of K, two of V

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r16 = lane & 15, g4 = lane >> 4, group = wave / SG, half = wave % SG;
  const int blocks = (a.G * a.Sq + BR - 1) / BR;
  const Slot slot = slot_of(a, id, blocks);
  const int bh = slot.bh, blk = blocks - 1 - slot.blk;
  const Rows w = rows_of(a, bh);
  const int rows = a.G * w.lq;
  const int r_wave = blk * BR + group * 32;
  const int last_row = min(blk * BR + BR, rows) - 1;
  int keys = 0;
  if (last_row >= blk * BR) keys = a.causal ? min(w.lk, query_of(a, last_row) + w.off + 1) : w.lk;
  const int tiles = keys > 0 ? (keys + TILE - 1) / TILE : 0;

  const unsigned short *Kg = slice(a.k, w.b, w.hk), *Vg = slice(a.v, w.b, w.hk);
  auto request = [&](int t) __attribute__((always_inline)) {
    const int left = w.lk - t * TILE, at = (t & 1) * T::BYTES, lane_ = fresh(lane);
    const unsigned kss = (unsigned)a.k.ss * 2u, vss = (unsigned)a.v.ss * 2u;
    const unsigned short *kt = Kg + (long long)t * TILE * a.k.ss, *vt = Vg + (long long)t * TILE * a.v.ss;
    if (left >= TILE) {
      constexpr int STEP = WAVES * 64 / T::CH;
      load_tile<DL, WAVES>(kt, (long long)kss * STEP, sK + at, a.D, lane_, wave, [&](int row) { return row * kss; });
      load_tile<DL, WAVES>(vt, (long long)vss * STEP, sK + V_AT + at, a.D, lane_, wave, [&](int row) { return row * vss; });
    } else {
      load_tile_any<DL, WAVES>(kt, sK + at, a.D, lane_, wave, [&](int row) { return row < left ? row * kss : BEYOND; });
      load_tile_any<DL, WAVES>(vt, sK + V_AT + at, a.D, lane_, wave, [&](int row) { return row < left ? row * vss : BEYOND; });
    }
  };
  if (tiles > 0) request(0);  // (in flight while the rest is set up)

  int q_last[2];
  float nl[2], nd[2];
  u32x4 qf[2][KS], of[2][KS];
#pragma unroll
  for (int qb = 0; qb < 2; ++qb) {
    const int r = r_wave + qb * 16 + r16;
    const bool there = r < rows;
    q_last[qb] = !there ? -1 : a.causal ? min(w.lk - 1, query_of(a, r) + w.off) : w.lk - 1;
    // (a row that sees one key has P = 1 whatever the score: no gradient, not the rounding of O in delta)
    if (q_last[qb] == 0) q_last[qb] = -1;
    const unsigned short *p = (const unsigned short *)a.q.p + (there ? row_at(a, a.q, w, r) : 0);
    const unsigned short *g = (const unsigned short *)a.d_o.p + (there ? row_at(a, a.d_o, w, r) : 0);
    nl[qb] = there ? a.neg_lse2[(long long)bh * a.rows_pad + r] : -INFINITY;
    nd[qb] = there ? a.neg_delta[(long long)bh * a.rows_pad + r] : 0.0f;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      qf[qb][ks] = resident(p, there, ks * 32 + g4 * 8, a.D);
      if (a.negate) qf[qb][ks] ^= 0x80008000u;
      of[qb][ks] = resident(g, there, ks * 32 + g4 * 8, a.D);
    }
  }
  int wave_keys = 0, wave_full = 0;
  if (r_wave < rows) {
    const int r_end = min(r_wave + 32, rows) - 1;
    wave_keys = a.causal ? min(w.lk, query_of(a, r_end) + w.off + 1) : w.lk;
    wave_full = a.causal ? min(w.lk, query_of(a, r_wave) + w.off + 1) : w.lk;  // (rows past the end have P = 0)
  }
  float dsc = 1.0f, dsp = 1.0f;  // dS operand = P' (dP - delta) dsp = dS dsc
  if constexpr (DT == DT_F16) {
    dsc = ds_scale(a, bh, lane);
    dsp = dsc * (1.0f / 16384.0f);
  }


  f32x4 acc[2][DB];
#pragma unroll
  for (int qb = 0; qb < 2; ++qb)
#pragma unroll
    for (int d = 0; d < DB; ++d) acc[qb][d] = f32x4{0, 0, 0, 0};

  const unsigned rows0 = rows_base<DL>(sK, r16, g4), cols0 = columns_base<DL>(sK, r16, g4);
  // A tile's first-operand fragments in the order of their use, for half-tiles s = 0, 1: S, dP (under it the exponentials of S),
  // then S of the other half (under it this half's dS), its dP, and dQ of both.  One chunk per fragment: the read of the fragment AHEAD chunks
  // on, the two products of this one, a share of the vector work.
  auto compute = [&](int t, auto edge_tag) __attribute__((always_inline)) {
    constexpr bool EDGE = decltype(edge_tag)::value;
    constexpr int AHEAD = 2, PER = (16 + DB - 1) / DB, H = 2 / SG, N = 3 * DB * H;
    const unsigned at_r = rows0 + (unsigned)(t & 1) * T::BYTES, at_c = cols0 + (unsigned)(t & 1) * T::BYTES;
    f32x4 z[H][2][2], g[2][2];  // [half][qb][block of 16 keys]
    u32x4 df[2], frag[AHEAD + 1];
    // phase of chunk i: S 0, dP 1, dQ 2 of half h
    auto phase = [](int i) constexpr { return H == 1 ? i / DB : (i / DB == 0 || i / DB == 2) ? 0 : (i / DB == 1 || i / DB == 3) ? 1 : 2; };
    auto half_of = [](int i) constexpr { return H == 1 ? 0 : i / DB < 2 ? 0 : i / DB < 4 ? 1 : i / DB - 4; };
    auto read = [&](auto tag) __attribute__((always_inline)) {
      constexpr int i = decltype(tag)::value, j = i % DB;
      if constexpr (i < N) {
        const int s = SG == 1 ? half_of(i) : half;
        if constexpr (phase(i) == 0) frag[i % (AHEAD + 1)] = read_rows<DL>(at_r, 0, 2 * s + j % 2, j / 2);
        else if constexpr (phase(i) == 1) frag[i % (AHEAD + 1)] = read_rows<DL>(at_r, V_AT, 2 * s + j % 2, j / 2);
        else frag[i % (AHEAD + 1)] = read_columns<DL>(at_c, 0, s, j);
      }
    };
    auto probability = [&](int h, int v) __attribute__((always_inline)) {
      const int qb = v >> 3, kb = (v >> 2) & 1, e = v & 3, s = SG == 1 ? h : half;
      float p = __builtin_amdgcn_exp2f(__builtin_fmaf(z[h][qb][kb][e], a.scale_log2, nl[qb]));
      if constexpr (EDGE) p = t * TILE + s * 32 + kb * 16 + g4 * 4 + e > q_last[qb] ? 0.0f : p;
      if constexpr (DT == DT_F16) p *= dsp;
      z[h][qb][kb][e] = p;
    };
    auto gradient = [&](int h, int v) __attribute__((always_inline)) {
      const int qb = v >> 3, kb = (v >> 2) & 1, e = v & 3;
      z[h][qb][kb][e] *= g[qb][kb][e];
    };
    u32x4 df1[2];  // of half 0 while half 1 is under way
    static_for<0, AHEAD>([&](auto tag) __attribute__((always_inline)) { read(tag); });
    static_for<0, N>([&](auto tag) __attribute__((always_inline)) {
      constexpr int i = decltype(tag)::value, j = i % DB, kb = j % 2, ks = j / 2, h = half_of(i), ph = phase(i);
      const u32x4 &f = frag[i % (AHEAD + 1)];
      read(std::integral_constant<int, i + AHEAD>{});
#pragma unroll
      for (int qb = 0; qb < 2; ++qb) {
        if constexpr (ph == 0) z[h][qb][kb] = Mfma16<DT>::run(f, qf[qb][ks], ks == 0 ? f32x4{0, 0, 0, 0} : z[h][qb][kb]);
        else if constexpr (ph == 1) g[qb][kb] = Mfma16<DT>::run(f, of[qb][ks], ks == 0 ? f32x4{nd[qb], nd[qb], nd[qb], nd[qb]} : g[qb][kb]);
        else acc[qb][j] = Mfma16<DT>::run(f, H == 2 && h == 0 ? df1[qb] : df[qb], acc[qb][j]);
      }
#pragma unroll
      for (int v = j * PER; v < j * PER + PER && v < 16; ++v) {
        if constexpr (ph == 1) probability(h, v);
        if constexpr (H == 2 && i / DB == 2) gradient(0, v);
        if constexpr (H == 2 && i / DB == 4) gradient(1, v);
      }
      if constexpr (H == 2 && i == 3 * DB - 1) {
#pragma unroll
        for (int qb = 0; qb < 2; ++qb) df1[qb] = pack_operand<DT>(z[0][qb][0], z[0][qb][1]);
      }
      if constexpr (H == 2 && i == 5 * DB - 1) {
#pragma unroll
        for (int qb = 0; qb < 2; ++qb) df[qb] = pack_operand<DT>(z[H - 1][qb][0], z[H - 1][qb][1]);
      }
      if constexpr (H == 1 && i == 2 * DB - 1) {
#pragma unroll
        for (int v = 0; v < 16; ++v) gradient(0, v);
#pragma unroll
        for (int qb = 0; qb < 2; ++qb) df[qb] = pack_operand<DT>(z[0][qb][0], z[0][qb][1]);
      }
      fence();
    });
  };
  auto head = [&](int t) __attribute__((always_inline)) {
    __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0): this tile
    __syncthreads();
    if (t + 1 < tiles) request(t + 1);
  };
  // tiles that every row of the wave sees whole, then the others (a wave takes part in the loads of tiles that none sees)
  int t = 0;
  for (const int end = min(tiles, wave_full / TILE); t < end; ++t) {
    head(t);
    compute(t, std::false_type{});
  }
  for (; t < tiles; ++t) {
    head(t);
    if (t * TILE < wave_keys) compute(t, std::true_type{});
  }

  if constexpr (SG == 2) join_halves<2 * DB>(sK, group, half, lane, [&](int i) -> f32x4 & { return acc[i / DB][i % DB]; });
  if (half != 0) return;
  const float f = (a.negate ? -a.scale : a.scale) / dsc;
#pragma unroll
  for (int qb = 0; qb < 2; ++qb) {
    const int r = r_wave + qb * 16 + r16;
    if (r >= a.G * a.Sq) continue;
    unsigned short *p = (unsigned short *)a.dq.p + row_at(a, a.dq, w, r);
#pragma unroll
    for (int d = 0; d < DB; ++d)
      if (d * 16 + g4 * 4 < a.D) *(u32x2 *)(p + d * 16 + g4 * 4) = pack_result<DT>(acc[qb][d], f);
  }
}

// dK and dV of a block of keys, or of a part of the rows that see them: four products per tile.  SG = 2: two waves share 32 keys,
// each takes half of every tile of rows.
template <int DT, int DL, int DU, int WAVES, int SG>
__device__ __forceinline__ void dkv_block(const AttentionTrainArgs &a, int id, unsigned char *sQ, float *sL, float *sD, u32x4 *parked) {
  using T = Tile<DL>;
  constexpr int BC = 32 * WAVES / SG, KS = DU / 32, DB = DU / 16;
  constexpr unsigned O_AT = 2 * T::BYTES;  // two tiles of Q, two of dO

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r16 = lane & 15, g4 = lane >> 4, group = wave / SG, half = wave % SG;
  const int blocks = (a.Sk + BC - 1) / BC;
  const Slot slot = slot_of(a, id, blocks * a.row_splits);
  const int bh = slot.bh, blk = slot.blk / a.row_splits, part = slot.blk - blk * a.row_splits;  // (causal: the first keys have most rows)
  const Rows w = rows_of(a, bh);
  const int rows = a.G * w.lq;
  const int k_blk = blk * BC, k_wave = k_blk + group * 32;

  // tiles of packed rows that see a key of the block, from the first one on
  int t_begin = a.causal ? (int)(((long long)max(0, k_blk - w.off) * a.G) / TILE) : 0;
  int t_end = k_blk < w.lk ? (rows + TILE - 1) / TILE : 0;
  if (a.row_splits > 1) {
    const int n = max(0, t_end - t_begin), from = t_begin;
    t_begin = from + n * part / a.row_splits;
    t_end = from + n * (part + 1) / a.row_splits;
  }

  const unsigned short *Qg = slice(a.q, w.b, w.hk * a.G), *Og = slice(a.d_o, w.b, w.hk * a.G);
  const float *nl = a.neg_lse2 + (long long)bh * a.rows_pad, *nd = a.neg_delta + (long long)bh * a.rows_pad;
  auto request = [&](int t) __attribute__((always_inline)) {
    const int r0 = t * TILE, i0 = query_of(a, r0), at = (t & 1) * T::BYTES, lane_ = fresh(lane);
    const unsigned short *qt = Qg + (long long)i0 * a.q.ss, *ot = Og + (long long)i0 * a.d_o.ss;
    auto offset = [&](const HeadView &v, int row) __attribute__((always_inline)) -> unsigned {
      const int r = r0 + row, i = query_of(a, r);
      return (unsigned)(i - i0) * ((unsigned)v.ss * 2u) + (unsigned)(r - i * a.G) * ((unsigned)v.sh * 2u);
    };
    constexpr int STEP = WAVES * 64 / T::CH;
    if (r0 + TILE <= rows && 16 % a.G == 0) {  // (a power of two: rows 16 apart are 16 / G queries apart)
      load_tile<DL, WAVES>(qt, (long long)(STEP / a.G) * a.q.ss * 2, sQ + at, a.D, lane_, wave, [&](int row) { return offset(a.q, row); });
      load_tile<DL, WAVES>(ot, (long long)(STEP / a.G) * a.d_o.ss * 2, sQ + O_AT + at, a.D, lane_, wave, [&](int row) { return offset(a.d_o, row); });
    } else {
      load_tile_any<DL, WAVES>(qt, sQ + at, a.D, lane_, wave, [&](int row) { return r0 + row < rows ? offset(a.q, row) : BEYOND; });
      load_tile_any<DL, WAVES>(ot, sQ + O_AT + at, a.D, lane_, wave, [&](int row) { return r0 + row < rows ? offset(a.d_o, row) : BEYOND; });
    }
    if (wave < 2) {  // (rows_pad is a multiple of the tile)
      dma4(resource((wave == 0 ? nl : nd) + r0, TILE * 4), lane * 4, lds_address((wave == 0 ? sL : sD) + (t & 1) * TILE));
    }
  };
  if (t_begin < t_end) request(t_begin);  // (in flight while the rest is set up)

  u32x4 kf[2][KS], vf[2][KS];
#pragma unroll
  for (int nb = 0; nb < 2; ++nb) {
    const int j = k_wave + nb * 16 + r16;
    const bool there = j < w.lk;
    const unsigned short *kp = slice(a.k, w.b, w.hk) + (there ? (long long)j * a.k.ss : 0);
    const unsigned short *vp = slice(a.v, w.b, w.hk) + (there ? (long long)j * a.v.ss : 0);
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      kf[nb][ks] = resident(kp, there, ks * 32 + g4 * 8, a.D);
      if (a.negate) kf[nb][ks] ^= 0x80008000u;
      vf[nb][ks] = resident(vp, there, ks * 32 + g4 * 8, a.D);
    }
  }
  // (D = 128 is some registers short: three fragments wait in LDS; a fourth would cost the second workgroup of a CU)
  constexpr bool PARK = DU == 128;
  auto own = [&](int i) -> u32x4 & { return parked[(wave * 3 + i) * 64 + (int)fresh(lane)]; };
  if constexpr (PARK) {
    own(0) = vf[0][KS - 1];
    own(1) = vf[1][KS - 1];
    own(2) = kf[1][KS - 1];
  }
  // of the wave: rows from here on see some of its keys / all of them (rows past the end have P = 0)
  const bool live = k_wave < w.lk;
  long long row_some = 0, row_all = 0;
  if (a.causal) {
    row_some = (long long)max(0, k_wave - w.off) * a.G;
    row_all = (long long)max(0, k_wave + 31 - w.off) * a.G;
  }
  if (w.lk == 1) row_all = 0x7fffffff;
  // The first packed row that sees the lane's key of block 0 (block 1: first_step further); and the first row that sees more than
  // one key: a row that sees one has P = 1 whatever the score, and no gradient (not the rounding of O in delta).
  const int first_row = a.causal ? (k_wave + r16 - w.off) * a.G : 0, first_step = a.causal ? 16 * a.G : 0;
  const int two_keys = w.lk == 1 ? 0x7fffffff : a.causal ? (1 - w.off) * a.G : 0;
  float dsc = 1.0f, dsp = 1.0f;
  if constexpr (DT == DT_F16) {
    dsc = ds_scale(a, bh, lane);
    dsp = dsc * (1.0f / 16384.0f);
  }


  f32x4 dk[2][DB], dv[2][DB];
#pragma unroll
  for (int nb = 0; nb < 2; ++nb)
#pragma unroll
    for (int d = 0; d < DB; ++d) dk[nb][d] = dv[nb][d] = f32x4{0, 0, 0, 0};

  auto compute = [&](int t, auto edge_tag) __attribute__((always_inline)) {
    constexpr bool EDGE = decltype(edge_tag)::value;
    const int lane_ = fresh(lane);
    const unsigned rows_at = rows_base<DL>(sQ, lane_ & 15, lane_ >> 4) + (unsigned)(t & 1) * T::BYTES;
    const unsigned cols_at = columns_base<DL>(sQ, lane_ & 15, lane_ >> 4) + (unsigned)(t & 1) * T::BYTES;
    const float *tL = sL + (t & 1) * TILE, *tD = sD + (t & 1) * TILE;
#pragma unroll
    for (int n = 0; n < 2 / SG; ++n) {
      const int s = SG == 1 ? n : half;
      // S; dP with the exponentials of S under it; dV with dS under it; dK.  One chunk per first-operand fragment: the read of the
      // fragment AHEAD chunks on, the two products of this one, a share of the vector work.
      constexpr int AHEAD = DU == 128 ? 1 : 2, PER = (16 + DB - 1) / DB, N = 4 * DB;
      f32x4 z[2][2], g[2][2], l4, d4[2];  // [block of 16 rows][nb]
      u32x4 pf[2], frag[AHEAD + 1];  // (dS takes P's place once dV has it)
      const unsigned at_r = fresh(rows_at), at_c = fresh(cols_at);
      auto read = [&](auto tag) __attribute__((always_inline)) {
        constexpr int i = decltype(tag)::value, j = i % DB;
        if constexpr (i < DB) frag[i % (AHEAD + 1)] = read_rows<DL>(at_r, 0, 2 * s + j % 2, j / 2);
        else if constexpr (i < 2 * DB) frag[i % (AHEAD + 1)] = read_rows<DL>(at_r, O_AT, 2 * s + j % 2, j / 2);
        else if constexpr (i < 3 * DB) frag[i % (AHEAD + 1)] = read_columns<DL>(at_c, O_AT, s, j);
        else if constexpr (i < N) frag[i % (AHEAD + 1)] = read_columns<DL>(at_c, 0, s, j);
      };
      static_for<0, AHEAD>([&](auto tag) __attribute__((always_inline)) { read(tag); });
      static_for<0, N>([&](auto tag) __attribute__((always_inline)) {
        constexpr int i = decltype(tag)::value, phase = i / DB, j = i % DB, rb = j % 2, ks = j / 2;
        const u32x4 &f = frag[i % (AHEAD + 1)];
        read(std::integral_constant<int, i + AHEAD>{});
        if constexpr (i == DB - 1) {
          d4[0] = *(const f32x4 *)(tD + s * 32 + g4 * 4);
          d4[1] = *(const f32x4 *)(tD + s * 32 + 16 + g4 * 4);
          l4 = *(const f32x4 *)(tL + s * 32 + g4 * 4);
        }
#pragma unroll
        for (int nb = 0; nb < 2; ++nb) {
          if constexpr (phase == 0) z[rb][nb] = Mfma16<DT>::run(f, PARK && nb == 1 && ks == KS - 1 ? own(2) : kf[nb][ks], ks == 0 ? f32x4{0, 0, 0, 0} : z[rb][nb]);
          else if constexpr (phase == 1) g[rb][nb] = Mfma16<DT>::run(f, PARK && ks == KS - 1 ? own(nb) : vf[nb][ks], ks == 0 ? d4[rb] : g[rb][nb]);
          else if constexpr (phase == 2) dv[nb][j] = Mfma16<DT>::run(f, pf[nb], dv[nb][j]);
          else dk[nb][j] = Mfma16<DT>::run(f, pf[nb], dk[nb][j]);
        }
        int limit[2];  // of the lane's key: rows of this half-tile below it do not count
        if constexpr (EDGE) {
#pragma unroll
          for (int nb = 0; nb < 2; ++nb) {
            const int from = (int)fresh(first_row) + nb * first_step;
            limit[nb] = (phase == 2 ? max(from, two_keys) : from) - (t * TILE + s * 32 + g4 * 4);
          }
        }
#pragma unroll
        for (int v = j * PER; v < j * PER + PER && v < 16; ++v) {
          const int vr = v >> 3, nb = (v >> 2) & 1, e = v & 3;
          if constexpr (phase == 1) {
            if (v == 8) l4 = *(const f32x4 *)(tL + s * 32 + 16 + g4 * 4);
            float p = __builtin_amdgcn_exp2f(__builtin_fmaf(z[vr][nb][e], a.scale_log2, l4[e]));
            if constexpr (EDGE) p = vr * 16 + e < limit[nb] ? 0.0f : p;
            z[vr][nb][e] = p;
          } else if constexpr (phase == 2) {
            float x = z[vr][nb][e] * g[vr][nb][e];
            if constexpr (DT == DT_F16) x *= dsp;
            if constexpr (EDGE) x = vr * 16 + e < limit[nb] ? 0.0f : x;
            z[vr][nb][e] = x;
          }
        }
        if constexpr (i == 2 * DB - 1 || i == 3 * DB - 1) {
#pragma unroll
          for (int nb = 0; nb < 2; ++nb) pf[nb] = pack_operand<DT>(z[0][nb], z[1][nb]);
        }
        fence();
      });
    }
  };
  auto head = [&](int t) __attribute__((always_inline)) {
    __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0): this tile
    __syncthreads();
    if (t + 1 < t_end) request(t + 1);
  };
  // tiles with rows that see some of the wave's keys, then those whose rows see all
  int t = t_begin;
  for (; t < t_end && t * TILE < row_all; ++t) {
    head(t);
    if (live && t * TILE + TILE > row_some) compute(t, std::true_type{});
  }
  for (; t < t_end; ++t) {
    head(t);
    if (live) compute(t, std::false_type{});
  }

  if constexpr (SG == 2)
    join_halves<4 * DB>(sQ, group, half, lane, [&](int i) -> f32x4 & { return i < 2 * DB ? dk[i / DB][i % DB] : dv[i / DB - 2][i % DB]; });
  if (half != 0) return;
  const float fk = (a.negate ? -a.scale : a.scale) / dsc, fv = DT == DT_F16 ? 1.0f / 16384.0f : 1.0f;
#pragma unroll
  for (int nb = 0; nb < 2; ++nb) {
    const int j = k_wave + nb * 16 + r16;
    if (j >= a.Sk) continue;
    unsigned short *kp = (unsigned short *)slice(a.dk, w.b, w.hk) + (long long)j * a.dk.ss;
    unsigned short *vp = (unsigned short *)slice(a.dv, w.b, w.hk) + (long long)j * a.dv.ss;
    const bool there = j < w.lk;  // (a key past the end was read as zeros, its P is not)
    if (a.row_splits > 1) {
      float *at = a.part_dkv + (((long long)part * a.B * a.Hk + bh) * a.Sk + j) * 2 * DU + g4 * 4;
#pragma unroll
      for (int d = 0; d < DB; ++d)
        if (there && d * 16 + g4 * 4 < a.D) {  // (what lies behind the length is not read)
          *(f32x4 *)(at + d * 16) = dk[nb][d] * fk;
          *(f32x4 *)(at + DU + d * 16) = dv[nb][d] * fv;
        }
      continue;
    }
#pragma unroll
    for (int d = 0; d < DB; ++d)
      if (d * 16 + g4 * 4 < a.D) {
        u32x2 x = pack_result<DT>(dk[nb][d], fk), y = pack_result<DT>(dv[nb][d], fv);
        *(u32x2 *)(kp + d * 16 + g4 * 4) = there ? x : u32x2{0, 0};
        *(u32x2 *)(vp + d * 16 + g4 * 4) = there ? y : u32x2{0, 0};
      }
  }
}

// The workgroups of dK and dV first, then those of dQ: one launch, so that neither waits for the other's last ones.
// Bound, long rows: matrix pipe and vector work of two waves per SIMD, and power: B4 H32 S4096 D128 bf16 3.05-3.15 ms =
// 1.22-1.26 PFLOP/s of the seven products, 0.87-0.90 of the five that are needed.  Short rows: the walk of a workgroup over its tiles
// one after another, each waited for whole, B1 H12 S1024 D64 f16 causal 23 us, S197 11 us: 0.95 us a tile of 64 by the plan's fit, of which
// its products are 0.2 us of the matrix pipe.
template <int DT, int DL, int DU, int WAVES, int SG>
__global__ void __launch_bounds__(WAVES * 64) __attribute__((amdgpu_waves_per_eu(2, 2)))
attention_train_backward_kernel(const AttentionTrainArgs a, int dkv_blocks) {
  __shared__ __attribute__((aligned(1024))) unsigned char tiles[4 * Tile<DL>::BYTES];
  __shared__ __attribute__((aligned(16))) float sL[2 * TILE], sD[2 * TILE];
  __shared__ u32x4 parked[DU == 128 ? WAVES * 3 * 64 : 1];
  if ((int)blockIdx.x < dkv_blocks) dkv_block<DT, DL, DU, WAVES, SG>(a, blockIdx.x, tiles, sL, sD, parked);
  else dq_block<DT, DL, DU, WAVES, SG>(a, blockIdx.x - dkv_blocks, tiles);
}

// Adds up the parts of dK and dV where the rows are split over workgroups, in their order: 4 columns per thread.  Bound by reading the
// parts: 9.3 us for two parts of B4 H4 S1500 D96 (46 MB with the results, 5.0 TB/s).
template <int DT, int DU>
__global__ void __launch_bounds__(256) attention_train_sum_kernel(const AttentionTrainArgs a) {
  constexpr int PER = 2 * DU / 4;
  const long long id = (long long)blockIdx.x * 256 + threadIdx.x, key = id / PER;
  const int piece = (int)(id - key * PER), c = (piece % (DU / 4)) * 4;
  const bool is_v = piece >= DU / 4;
  if (key >= (long long)a.B * a.Hk * a.Sk || c >= a.D) return;
  const int bh = (int)(key / a.Sk), j = (int)(key - (long long)bh * a.Sk), b = bh / a.Hk;
  const long long plane = (long long)a.B * a.Hk * a.Sk * 2 * DU;
  const float *at = a.part_dkv + key * 2 * DU + piece * 4;
  f32x4 x = {0, 0, 0, 0};
  if (j < rows_of(a, bh).lk) {
    x = *(const f32x4 *)at;
    for (int r = 1; r < a.row_splits; ++r) x += *(const f32x4 *)(at + r * plane);
  }
  const HeadView &out = is_v ? a.dv : a.dk;
  *(u32x2 *)((unsigned short *)slice(out, b, bh - b * a.Hk) + (long long)j * out.ss + c) = pack_result<DT>(x, 1.0f);
}

template <int DT, int DL, int DU>
int forward(const AttentionTrainArgs &a, hipStream_t stream) {
  constexpr int W = 4;
  const dim3 grid((unsigned)((a.G * a.Sq + a.block - 1) / a.block) * (unsigned)(a.B * a.Hk), (unsigned)a.splits);
  if (a.block == 32 * W) hipLaunchKernelGGL((attention_train_forward_kernel<DT, DL, DU, W, 1, 2>), grid, dim3(W * 64), 0, stream, a);
  else if (a.block == 16 * W) hipLaunchKernelGGL((attention_train_forward_kernel<DT, DL, DU, W, 2, 2>), grid, dim3(W * 64), 0, stream, a);
  else hipLaunchKernelGGL((attention_train_forward_kernel<DT, DL, DU, W, 2, 1>), grid, dim3(W * 64), 0, stream, a);
  if (a.splits > 1) {
    const long long rows = (long long)a.B * a.Hk * a.G * a.Sq;
    hipLaunchKernelGGL((attention_train_join_kernel<DT, DU>), dim3((unsigned)((rows + 7) / 8)), dim3(256), 0, stream, a);
  }
  return (int)hipGetLastError();
}

template <int DT, int DL, int DU>
int backward(const AttentionTrainArgs &a, hipStream_t stream) {
  constexpr int W = 4;
  const unsigned bh = (unsigned)(a.B * a.Hk);
  const unsigned row_blocks = (unsigned)(DT == DT_F16 ? a.norm_blocks : a.rows_pad / TILE);
  if (row_blocks > 0) hipLaunchKernelGGL((attention_train_rows_kernel<DT>), dim3(row_blocks * bh), dim3(256), 0, stream, a);
  auto blocks = [&](int n) { return (unsigned)((n + a.block - 1) / a.block) * bh; };
  const unsigned kb = blocks(a.Sk) * (unsigned)a.row_splits, qb = blocks(a.G * a.Sq);
  if (kb + qb > 0) {
    if (a.block == 32 * W) hipLaunchKernelGGL((attention_train_backward_kernel<DT, DL, DU, W, 1>), dim3(kb + qb), dim3(W * 64), 0, stream, a, (int)kb);
    else hipLaunchKernelGGL((attention_train_backward_kernel<DT, DL, DU, W, 2>), dim3(kb + qb), dim3(W * 64), 0, stream, a, (int)kb);
  }
  if (a.row_splits > 1 && a.Sk > 0) {
    const long long pieces = (long long)a.B * a.Hk * a.Sk * 2 * DU / 4;
    hipLaunchKernelGGL((attention_train_sum_kernel<DT, DU>), dim3((unsigned)((pieces + 255) / 256)), dim3(256), 0, stream, a);
  }
  return (int)hipGetLastError();
}

template <int DT>
int forward_any(const AttentionTrainArgs &a, hipStream_t stream) {
  return a.D <= 64 ? forward<DT, 64, 64>(a, stream) : a.D <= 96 ? forward<DT, 128, 96>(a, stream) : forward<DT, 128, 128>(a, stream);
}
template <int DT>
int backward_any(const AttentionTrainArgs &a, hipStream_t stream) {
  return a.D <= 64 ? backward<DT, 64, 64>(a, stream) : a.D <= 96 ? backward<DT, 128, 96>(a, stream) : backward<DT, 128, 128>(a, stream);
}

}  // namespace

int launch_attention_train_forward(const AttentionTrainArgs &a, int dtype, hipStream_t stream) {
  return dtype == DT_F16 ? forward_any<DT_F16>(a, stream) : forward_any<DT_BF16>(a, stream);
}
int launch_attention_train_backward(const AttentionTrainArgs &a, int dtype, hipStream_t stream) {
  return dtype == DT_F16 ? backward_any<DT_F16>(a, stream) : backward_any<DT_BF16>(a, stream);
}

}  // namespace tracea_amd
