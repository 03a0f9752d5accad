// Attention over a key/value cache in pages for blocks of many rows (a piece of a prompt), gfx950.  The formulas are those of
// attention_cached_kernels.hip, the walk is that of the forward pass for training (attention_train_kernels.hip): a wave owns 32 rows whose
// queries stay in registers, tiles of 64 keys and values go through LDS, the scores of tile t + 1 are computed under the exponentials of tile t and
// P V of tile t under the maximum over t + 1, so that K is a tile ahead of V.
//
// A tile is four groups of 16 keys, each in one page: its requests take their rows' place from the group.  In 16 bits they go straight
// to LDS.  In 8 bits a thread keeps 8 codes of each of its rows in registers while the tile before is worked on, and widens them on
// their way to LDS once for the four waves, which then read what they would of a cache of 16 bits.
//
// Bound by the matrix pipe (busy for a third of the time) and the vector work beside it (exponentials, maxima, packing: half of the time), which
// two waves a SIMD overlap only in part.  1024 queries of 32:8 heads of 128 columns over 8192 keys, two sequences: 315 us in 8 bits (0.82
// PFLOP/s; the library's largest product reaches 1.27), 279 us in 16 (0.92); of unlike lengths (8192 and about 5000) 255 us in 8 bits on one set
// of operands, 280 to 286 on two in turn, and 217 in 16, as the shorter one leaves its places empty.
#include <type_traits>

#include "attention_cached_share.hpp"

namespace tracea_amd {

namespace {

constexpr int WAVES = 4, NQ = 2, KB = TILE / 16, ROWS = 16 * NQ * WAVES;

// The (sequence, head, block of rows) of a workgroup, in an order that begins with those that take longest: they are handed out as slots
// come free, and the first of them on every CU share it with the last ones.  Where a sequence may have more than twice as many keys as queries
// its length decides (up to 64 sequences), then, or else, what a causal mask leaves of it.  Neighbours are different heads, so that a head stays on
// one XCD where there are 8 of them.
__device__ __forceinline__ void place_of(const AttentionCachedArgs &a, int lane, int &b, int &hk, int &rb) {
  const int id = blockIdx.x;
  if (a.B <= 64) {
    const int own = lane < a.B ? keys_of(a, lane) : -1;
    int rank = 0, longest = 0;
    for (int i = 0; i < a.B; ++i) {
      const int other = __builtin_amdgcn_readlane(own, i);
      longest = max(longest, other);
      rank += other > own || (other == own && i < lane);
    }
    if (longest > 2 * a.Sq) {
      const int per = a.Hk * a.row_blocks, turn = id / per, rest = id - turn * per, blk = rest / a.Hk;
      b = __builtin_amdgcn_readfirstlane(__ffsll((long long)__ballot(lane < a.B && rank == turn)) - 1);
      hk = rest - blk * a.Hk;
      rb = a.row_blocks - 1 - blk;
      return;
    }
  }
  const int heads = a.B * a.Hk, blk = id / heads, bh = (id - blk * heads + blk) % heads;
  b = bh / a.Hk;
  hk = bh - b * a.Hk;
  rb = a.row_blocks - 1 - blk;
}

template <int DT, bool C8, int DL, int DU>
__global__ void __launch_bounds__(WAVES * 64) __attribute__((amdgpu_waves_per_eu(2, 2))) attention_cached_tiles_kernel(const AttentionCachedArgs a) {
  using T = Tile<DL>;
  constexpr int KS = DU / 32, DB = DU / 16, RPI = 64 / T::CH, NI = TILE / (RPI * WAVES);
  constexpr unsigned SIDE = T::BYTES, V_AT = 2 * SIDE;  // two tiles of K, two of V
  __shared__ __attribute__((aligned(1024))) unsigned char sK[4 * SIDE];

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r16 = lane & 15, g4 = lane >> 4;

  int b, hk, rb;
  place_of(a, lane, b, hk, rb);
  const int lk = keys_of(a, b), lq = queries_of(a, b);
  const int rows = a.G * lq, off = lk - lq, r_wave = rb * ROWS + wave * 16 * NQ;

  const int last_row = min(rb * ROWS + ROWS, rows) - 1;
  int keys = 0;  // that any row of the block sees
  if (last_row >= rb * ROWS) keys = a.causal ? min(lk, query_of(a, last_row) + off + 1) : lk;
  int steps = keys > 0 ? (keys + TILE - 1) / TILE : 0, s0 = 0;
  const long long problem = ((long long)b * a.Hk + hk) * a.row_blocks + rb;
  bool cut = false;
  if (gridDim.y > 1) {  // the problem's steps in even parts
    const int per = max(1, (steps + (int)gridDim.y - 1) / (int)gridDim.y), parts = max(1, (steps + per - 1) / per);
    cut = parts > 1;
    if (blockIdx.y == 0 && threadIdx.x == 0) {
      a.meta[2 * problem] = cut ? (int)(problem * gridDim.y) : -1;
      a.meta[2 * problem + 1] = parts;
    }
    if ((int)blockIdx.y >= parts) return;
    s0 = (int)blockIdx.y * per;
    steps = min(steps, s0 + per);
  }

  f32x4 o[NQ][DB];
  float m[NQ];
  double total[NQ];
#pragma unroll
  for (int qb = 0; qb < NQ; ++qb) {
    m[qb] = -INFINITY;
    total[qb] = 0.0;
#pragma unroll
    for (int d = 0; d < DB; ++d) o[qb][d] = f32x4{0, 0, 0, 0};
  }

  Places at;  // of 16 tiles
  unsigned long long valid_before = 0;  // of the 16 before
  int located = 0;                      // the first of them
  // Scales of 8 bits: codes are widened with the power of two in their page's scale, which costs nothing and rounds nothing, in units of the
  // largest that the workgroup meets where f16 would leave its range.  A scale that is no power of two is met by the slow way (see settle_any).
  float ks, vs, k_unit = 1.0f, v_unit = 1.0f;  // of the lane's group; units
  bool powers = true;
  if constexpr (C8) {
    float k_top = 0.0f, v_top = 0.0f;
    unsigned odd = 0;
    const int end = min(lk, steps * TILE), first = s0 * TILE / a.table.P, last = end > s0 * TILE ? (end - 1) / a.table.P : first - 1;
    for (int i = first + lane; i <= last; i += 64) {
      const int page = page_of(a.table, b, i);
      if (page < 0) continue;
      const float x = a.ks.p[page * a.ks.sn + hk * a.ks.sh], y = a.vs.p[page * a.vs.sn + hk * a.vs.sh];
      k_top = fmaxf(k_top, x);
      v_top = fmaxf(v_top, y);
      odd |= (__builtin_bit_cast(unsigned, x) | __builtin_bit_cast(unsigned, y)) & 0x7fffffu;
    }
    powers = __ballot(odd != 0) == 0;
    if constexpr (DT == DT_F16) {
      k_unit = __builtin_bit_cast(float, max(__builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, wave_max(k_top))) & 0x7f800000, 0x00800000));
      v_unit = __builtin_bit_cast(float, max(__builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, wave_max(v_top))) & 0x7f800000, 0x00800000));
    }
  }
  const float c = fmaxf(a.scale_log2 * k_unit, 1.17549435e-38f);  // scores times it are exponents of 2 (above 0: -inf stays what it is)
  // Requests: a lane has 8 columns of one row of each.  A request's rows lie in one group of 16 keys, and a wave's requests are whole groups
  // apart, so that the lane's place in the group and its column are the same in all.
  constexpr int APART = WAVES * RPI;
  static_assert(APART % 16 == 0 && 16 % RPI == 0);
  const int my_row = wave * RPI + lane / T::CH, my_col = ((lane % T::CH) ^ T::swz(my_row)) << 3;
  const unsigned my_k = my_col >= a.D ? BEYOND : (unsigned)(my_row & 15) * (unsigned)a.k.ss + (unsigned)(my_col * (C8 ? 1 : 2));
  const unsigned my_v = my_col >= a.D ? BEYOND : (unsigned)(my_row & 15) * (unsigned)a.v.ss + (unsigned)(my_col * (C8 ? 1 : 2));
  u32x2 codes_k[C8 ? NI : 1], codes_v[C8 ? NI : 1];
  float scale_k[C8 ? NI : 1], scale_v[C8 ? NI : 1];  // of the groups whose codes are on their way
  auto request = [&](int tile, bool is_k, unsigned char *dst) __attribute__((always_inline)) {
    u32x2(&codes)[C8 ? NI : 1] = is_k ? codes_k : codes_v;
    auto go = [&](auto &&offset_of) __attribute__((always_inline)) {
      const unsigned lds = lds_address(dst);
#pragma unroll
      for (int i = 0; i < NI; ++i) {
        const int first = i * APART + wave * RPI, e = (tile & 15) * 4 + first / 16;
        const unsigned char *base = is_k ? at.k(e) : at.v(e);
        const unsigned offset = offset_of(i, e);
        if constexpr (C8) {
          (is_k ? scale_k : scale_v)[i] = of_lane(is_k ? ks : vs, e);
          codes[i] = __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(
                                                   __builtin_amdgcn_make_buffer_rsrc((void *)base, 0, (int)BEYOND, 0x00020000), (int)offset, 0, 0));
        } else {
          dma16(resource(base, BEYOND), offset, lds + (unsigned)(first * T::ROW_BYTES));
        }
      }
    };
    const unsigned mine = is_k ? my_k : my_v;
    if ((tile + 1) * TILE <= lk && ((unsigned)(at.valid >> (tile & 15) * 4) & 15u) == 15u)
      go([&](int, int) { return mine; });
    else  // rows without a key read as zeros
      go([&](int i, int e) { return tile * TILE + i * APART + my_row >= lk || !((at.valid >> e) & 1) ? BEYOND : mine; });
  };
  // Codes that have arrived, to where a request in 16 bits would have put them, times the power of two of their group's scale.
  auto settle_one = [&](unsigned char *dst, const u32x2 &codes, float scale, int i) __attribute__((always_inline)) {
    const float power = __builtin_bit_cast(float, __builtin_bit_cast(unsigned, scale) & 0x7f800000u);
    const u32x4 x = {widen2<DT, false>(codes[0], power), widen2<DT, true>(codes[0], power), widen2<DT, false>(codes[1], power),
                     widen2<DT, true>(codes[1], power)};
    *(u32x4 *)(dst + (i * APART + wave * RPI) * T::ROW_BYTES + lane * 16) = x;
  };
  // ... times any scale, rounded to the type of the products.
  auto settle_any = [&](unsigned char *dst, const u32x2 (&codes)[C8 ? NI : 1], const float (&scale)[C8 ? NI : 1]) __attribute__((always_inline)) {
    if constexpr (C8) {
#pragma unroll
      for (int i = 0; i < NI; ++i) {
        u32x4 x;
#pragma unroll
        for (int w = 0; w < 2; ++w) {
          x[2 * w] = pack2<DT>(__builtin_amdgcn_cvt_f32_fp8((int)codes[i][w], 0) * scale[i], __builtin_amdgcn_cvt_f32_fp8((int)codes[i][w], 1) * scale[i]);
          x[2 * w + 1] = pack2<DT>(__builtin_amdgcn_cvt_f32_fp8((int)codes[i][w], 2) * scale[i], __builtin_amdgcn_cvt_f32_fp8((int)codes[i][w], 3) * scale[i]);
        }
        *(u32x4 *)(dst + (i * APART + wave * RPI) * T::ROW_BYTES + lane * 16) = x;
      }
    }
  };
  auto settle = [&](unsigned char *dst, const u32x2 (&codes)[C8 ? NI : 1], const float (&scale)[C8 ? NI : 1]) __attribute__((always_inline)) {
    if constexpr (C8) {
#pragma unroll
      for (int i = 0; i < NI; ++i) settle_one(dst, codes[i], scale[i], i);
    }
  };
  auto locate = [&](int tile) __attribute__((always_inline)) {  // (a multiple of 16, or the first)
    valid_before = at.valid;
    located = tile & ~15;
    bool there;
    const int page = at.locate(a, b, hk, located * TILE + lane * 16, lk, there);
    if constexpr (C8) {
      // (a group without a page: 1, as its zeros stay zeros only with a finite scale, and that of a page that nobody uses may be anything)
      ks = there ? a.ks.p[page * a.ks.sn + hk * a.ks.sh] / k_unit : 1.0f;
      vs = there ? a.vs.p[page * a.vs.sn + hk * a.vs.sh] / v_unit : 1.0f;
    }
  };
  // Which groups of a tile in LDS have pages: the others' keys are zeros that nobody sees.
  auto valid_of = [&](int tile) { return (unsigned)((tile < located ? valid_before : at.valid) >> (tile & 15) * 4) & 15u; };
  auto k_side = [&](int tile) { return sK + (tile & 1) * SIDE; };
  auto v_side = [&](int tile) { return sK + V_AT + (tile & 1) * SIDE; };

  if (s0 < steps) {
    locate(s0);
    request(s0, true, k_side(s0));
    request(s0, false, v_side(s0));
  }

  int q_last[NQ];  // the last key that the lane's queries see
  u32x4 qf[NQ][KS];
#pragma unroll
  for (int qb = 0; qb < NQ; ++qb) {
    const int r = r_wave + qb * 16 + r16, i = query_of(a, r);
    const bool there = r < rows;
    q_last[qb] = !there ? -1 : a.causal ? min(lk - 1, i + off) : lk - 1;
    const unsigned short *p =
        (const unsigned short *)a.q.p + (there ? (long long)b * a.q.sb + (long long)(hk * a.G + r - i * a.G) * a.q.sh + (long long)i * a.q.ss : 0);
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) qf[qb][ks] = query_columns(a, p, there, ks * 32 + g4 * 8);
  }
  // of the wave: steps with a key that some row sees, and steps whose keys every row sees
  int wave_keys = 0, wave_full = 0;
  if (r_wave < rows) {
    const int r_end = min(r_wave + 16 * NQ, rows) - 1;
    wave_keys = a.causal ? min(lk, query_of(a, r_end) + off + 1) : lk;
    wave_full = a.causal ? min(lk, query_of(a, r_wave) + off + 1) : lk;  // (what rows past the end hold is dropped)
  }
  const int wave_steps = wave_keys > 0 ? min(steps, (wave_keys + TILE - 1) / TILE) : 0, full_steps = max(wave_full, 0) / TILE;

  const unsigned rows0 = rows_base<DL>(sK, r16, g4), cols0 = columns_base<DL>(sK, r16, g4);
  // What a row does not see becomes -inf; the largest score of the lane's in a tile, one value at a time.
  float block_max[NQ];
  auto take_max = [&](int step, int v, f32x4 (&z)[NQ][KB], float (&mx)[NQ], unsigned valid, auto edge_tag) __attribute__((always_inline)) {
    const int qb = v >> 4, kb = (v >> 2) & 3, e = v & 3;
    if constexpr (decltype(edge_tag)::value)
      z[qb][kb][e] = step * TILE + kb * 16 + g4 * 4 + e > q_last[qb] ? -INFINITY : z[qb][kb][e];
    block_max[qb] = e == 0 ? z[qb][kb][0] : fmaxf(block_max[qb], z[qb][kb][e]);
    if (e == 3) {
      mx[qb] = fmaxf(mx[qb], (valid >> kb) & 1u ? block_max[qb] : -INFINITY);
    }
  };
  // The rows' references, and what is summed up already, where a tile exceeds the scores they stand for by LAZY_MAX powers of two.
  auto move_reference = [&](const float (&mx)[NQ]) __attribute__((always_inline)) {
    bool moved = false;
    float alpha[NQ];
#pragma unroll
    for (int qb = 0; qb < NQ; ++qb) {
      const float top = groups_max_valu(mx[qb]) * c;
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
    const unsigned valid = valid_of(t), valid_next = valid_of(t + 1);
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
      const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(z[qb][kb][e], c, (valid >> kb) & 1u ? -ref[qb] : -INFINITY));
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
          for (int v = j * PER; v < (j + 1) * PER && v < 16 * NQ; ++v) take_max(t + 1, v, zn, mx, valid_next, edge_tag);
        }
      }
      // V of t + 1 and K of t + 2, where the products hide it (what was not requested goes where nobody reads any more)
      if constexpr (C8 && !LAST && i >= N - 2 * NI) {
        constexpr int p = i - (N - 2 * NI);
        if constexpr (p < NI) settle_one(v_side(t + 1), codes_v[p], scale_v[p], p);
        else settle_one(k_side(t + 2), codes_k[p - NI], scale_k[p - NI], p - NI);
      }
      fence();
    });
#pragma unroll
    for (int qb = 0; qb < NQ; ++qb) total[qb] += (double)sum[qb];
    if constexpr (!LAST) move_reference(mx);
  };
  // Step t: the scores of t are there; K of t + 1 and V of t have arrived, K of t + 2 and V of t + 1 go out.  (In their places K of t and V of
  // t - 1 were last read before the barrier.)
  auto head = [&](int t) __attribute__((always_inline)) {
    if constexpr (!C8) {
      __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0)
    } else if (!powers) {
      if (t > s0) settle_any(v_side(t), codes_v, scale_v);
      if (t + 1 < steps) settle_any(k_side(t + 1), codes_k, scale_k);
    }
    __syncthreads();
    if (t + 1 < steps) request(t + 1, false, v_side(t + 1));
    if (t + 2 < steps) {
      if (((t + 2) & 15) == 0) locate(t + 2);
      request(t + 2, true, k_side(t + 2));
    }
  };
  // ... of a wave that has no scores in step t + 1
  auto pass_on = [&](int t) __attribute__((always_inline)) {
    if (t + 1 < steps) settle(v_side(t + 1), codes_v, scale_v);
    if (t + 2 < steps) settle(k_side(t + 2), codes_k, scale_k);
  };

  f32x4 za[NQ][KB], zb[NQ][KB];
  int t = s0;
  if (t < steps) {
    __builtin_amdgcn_s_waitcnt(0x0f70);
    settle(k_side(t), codes_k, scale_k);
    settle(v_side(t), codes_v, scale_v);
    if (C8 && !powers) {
      settle_any(k_side(t), codes_k, scale_k);
      settle_any(v_side(t), codes_v, scale_v);
    }
    if (t + 1 < steps) {
      if (((t + 1) & 15) == 0) locate(t + 1);
      request(t + 1, true, k_side(t + 1));
    }
    __syncthreads();
    if (t < wave_steps) {  // the first scores, on their own
      const unsigned at_k = fresh(rows0) + (unsigned)(t & 1) * SIDE;
      float mx[NQ];
      const unsigned valid = valid_of(t);
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
      for (int v = 0; v < 16 * NQ; ++v) take_max(t, v, za, mx, valid, std::true_type{});
      move_reference(mx);
    }
    if (t + 1 < steps) settle(k_side(t + 1), codes_k, scale_k);
  }
  const int whole = min(full_steps, wave_steps) - 1, last = wave_steps - 1;  // steps whose next one is whole; the wave's last
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
    pass_on(t);
    ++t;
  }
  for (; t < steps; ++t) {  // (tiles that only other waves see)
    head(t);
    pass_on(t);
  }

  const long long slot = problem * gridDim.y + blockIdx.y;
  constexpr int WIDTH = DU <= 64 ? 64 : 128;
#pragma unroll
  for (int qb = 0; qb < NQ; ++qb) {
    const int row = wave * 16 * NQ + qb * 16 + r16, r = rb * ROWS + row;
    const float sum = groups_sum((float)total[qb]);
    if (r >= a.G * a.Sq) continue;
    if constexpr (C8) {
#pragma unroll
      for (int d = 0; d < DB; ++d) o[qb][d] *= v_unit;
    }
    if (cut) {
      if (g4 == 0) {
        a.part_ml[2 * (slot * ROWS + row)] = m[qb];
        a.part_ml[2 * (slot * ROWS + row) + 1] = sum;
      }
#pragma unroll
      for (int d = 0; d < DB; ++d)
        if (d * 16 + g4 * 4 < a.D) *(f32x4 *)(a.part_o + (slot * ROWS + row) * WIDTH + d * 16 + g4 * 4) = o[qb][d];
      continue;
    }
    const int i = query_of(a, r), h = hk * a.G + r - i * a.G;
    const bool there = r < rows && sum != 0.0f;  // a query of the sequence that sees a key
    const float inv = sum > 0.0f ? 1.0f / sum : sum;  // (NaN stays)
    unsigned short *p = (unsigned short *)a.o.p + (long long)b * a.o.sb + (long long)h * a.o.sh + (long long)i * a.o.ss;
#pragma unroll
    for (int d = 0; d < DB; ++d) {
      const int col = d * 16 + g4 * 4;
      if (col >= a.D) continue;
      u32x2 x = pack_result<DT>(o[qb][d], inv);
      if (!there) x = u32x2{0, 0};
      if (a.o_vec) {
        *(u32x2 *)(p + col) = x;
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) p[col + e] = (unsigned short)(x[e / 2] >> (e % 2 * 16));
      }
    }
    if (g4 == 0 && a.lse != nullptr)
      a.lse[(long long)b * a.lse_sb + (long long)h * a.lse_sh + (long long)i * a.lse_ss] = there ? (m[qb] + __builtin_amdgcn_logf(sum)) * LN2 : -INFINITY;
  }
}

template <int DT, int DL, int DU>
int launch(const AttentionCachedArgs &a, bool e4m3, hipStream_t stream) {
  const dim3 grid((unsigned)(a.B * a.Hk * a.row_blocks), (unsigned)a.splits), block(WAVES * 64);
  if (e4m3) hipLaunchKernelGGL((attention_cached_tiles_kernel<DT, true, DL, DU>), grid, block, 0, stream, a);
  else hipLaunchKernelGGL((attention_cached_tiles_kernel<DT, false, DL, DU>), grid, block, 0, stream, a);
  return (int)hipGetLastError();
}
template <int DT>
int launch_type(const AttentionCachedArgs &a, bool e4m3, hipStream_t stream) {
  if (a.D <= 64) return launch<DT, 64, 64>(a, e4m3, stream);
  return a.D <= 96 ? launch<DT, 128, 96>(a, e4m3, stream) : launch<DT, 128, 128>(a, e4m3, stream);
}

}  // namespace

int launch_attention_cached_tiles(const AttentionCachedArgs &a, int dtype, bool e4m3, hipStream_t stream) {
  return dtype == DT_F16 ? launch_type<DT_F16>(a, e4m3, stream) : launch_type<DT_BF16>(a, e4m3, stream);
}

}  // namespace tracea_amd
