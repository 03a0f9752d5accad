// Attention over a key/value cache in pages, gfx950: queries of a few rows against many keys in 16 bits, or in 8 with a scale for each page
// and head.
//
//   s_ij = scale q_i . k_j  over the keys a row sees     o_i = sum_j exp(s_ij - lse_i) v_j     lse_i = log sum_j exp(s_ij)
//   k_j = ks[page of j] code_j, v_j = vs[page of j] code_j: ks multiplies the score, vs the probability, both in fp32.
//
// Bound by reading the cache, once for each block of up to 32 rows: rows r = query G + head of the group are packed as in the attention for
// training, so that up to 32 heads and queries share a walk over the keys.  33 to 64 rows are two blocks, each with a walk of its own: 64:8 heads over 16
// sequences of 4096 keys, 4 queries (32 rows) 35 us in 8 bits, 5 to 8 queries 56; in 16 bits 52 and 81, where the tiles of 128 rows take 57 for 9.
// Nothing passes through LDS on its way: the products are v_mfma_f32_16x16x32, whose first operand is 8 values a lane, and which values these are
// is free as long as both operands agree.
//   S^T = K Q^T   of 16 keys: lane l has key l & 15 and the columns 8 KS (l >> 4) .. + 8 KS - 1, a run of the key's row; the resident
//                 queries are held by the same columns.  The result has row l & 15, keys 4 (l >> 4) + 0..3.
//   O^T += V^T P^T of 32 keys: with P as it lies, lane l's k slots are keys 4 (l >> 4) + 0..3 of both blocks of 16; it loads these 8 rows, of
//                 each the columns VC (l & 15) .. + VC - 1, and the product number j takes column j of each: a transposition by one byte
//                 permutation per two values.  The result has row l & 15 and, over the VC products, VC columns in a run for each of 4 lanes' chunks.
// Codes of 8 bits become f16 or bf16 exactly on the way (two per instruction).
//
// A wave walks every fourth block of 32 keys, the next one requested while it works on the last; a workgroup's four waves join through LDS.
// Where blocks of rows are few, all steps of 128 keys of all sequences are shared out evenly (attention_cached_share.hpp), whatever the
// lengths; a problem cut between workgroups is joined by a second launch, parts in their order.
//
// One query of 40:8 heads over 131072 keys of 128 columns in 8 bits (269 MB): 55 to 62 us, 4.3 to 4.9 TB/s (a copy: 5.06), 4 to 5 of them the second
// launch; 8 sequences of up to 8192 keys, 32:8 heads, 26 us (a copy: 18), of which 5 are a chain of dependent loads (lengths, table, keys, values)
// before the first result and 4 the second launch; 5 queries of 16:4 heads of 96 columns over 16 sequences of up to 2000 keys in 16 bits 18 us
// (a copy: 6.4), the same chain and three steps; one query of 12 heads over 197 keys 5.5 us, 8.6 where the table has room for 800 keys or more,
// as the plan is made for those.
#include <algorithm>
#include <type_traits>

#include "attention_cached_share.hpp"

namespace tracea_amd {

namespace {

constexpr int WAVES = 4;

// Of a cache in 8 bits, what the scales of the groups of 16 keys in Places make of scores and probabilities:
//   c     scale log2(e) ks: scores times c are exponents of 2 (above 0, so that -inf of a key that is not seen stays that)
//   lift  log2(vs / ref), ref the largest scale of values that the wave has met: what is summed up is in units of ref, so that f16
//         probabilities times a scale keep their range; the scale joins the probability in its exponent, p vs / ref = 2^(x - m + lift), and the sum
//         of probabilities takes it back, 2^-lift times a group's four.  -60 at least: less is nothing beside the largest.  The product is what is
//         rounded: below f16's normal numbers (a row's largest probability: lifts below -25) it is off by 2^-36 of ref.
constexpr float LEAST_LIFT = -60.0f;
struct Scales {
  float c, lift, ref = 0.0f;
  float lift_before;  // of the 64 groups before

  // The factor by which what is summed up so far changes.
  __device__ __forceinline__ float load(const AttentionCachedArgs &a, int hk, int page, bool there) {
    // (a group without a page: nothing of a scale that may be anything)
    const float ks = there ? a.ks.p[page * a.ks.sn + hk * a.ks.sh] : 1.0f, vs = there ? a.vs.p[page * a.vs.sn + hk * a.vs.sh] : 0.0f;
    c = fmaxf(a.scale_log2 * ks, 1.17549435e-38f);
    const float top = wave_max(vs);
    float f = 1.0f;
    lift_before = lift;
    if (top > ref) {  // (lifts from before, in its terms)
      f = ref / top;
      ref = top;
      lift_before = fmaxf(lift + fmaxf(__builtin_amdgcn_logf(f), LEAST_LIFT), LEAST_LIFT);
    }
    lift = fmaxf(__builtin_amdgcn_logf(vs / fmaxf(ref, 1.17549435e-38f)), LEAST_LIFT);
    return f;
  }
  __device__ __forceinline__ float unit() const { return fmaxf(ref, 1.17549435e-38f); }
};

template <int DT, bool C8, int DU, int NQ, bool FULL>
struct Stream {
  static constexpr int KS = DU / 32, VC = DU / 16, ES = C8 ? 1 : 2, ROWS = 16 * NQ;
  static constexpr int KW = 2 * ES, VW = VC * ES / 4;  // registers of 8 columns of a key, of a chunk of a row of values

  struct Keys {  // of a step: 32 keys
    unsigned k[2][KS][KW];
  };
  struct Values {
    unsigned v[8][VW];
  };
  struct Tags {
    unsigned valid;  // of the two groups of 16
    float c[2], lift[2];
  };
};

// Loads W registers from `base` (uniform) and a lane's offset, on 4, 8 or 16 bytes or less: the hardware takes 4.
template <int W>
__device__ __forceinline__ void load_words(const unsigned char *base, unsigned offset, unsigned (&to)[W]) {
  struct __attribute__((packed, aligned(4))) Words {
    unsigned w[W];
  };
  const Words x = *(const Words *)(base + offset);
#pragma unroll
  for (int i = 0; i < W; ++i) to[i] = x.w[i];
}

template <int DT, bool C8, int DU, int NQ, bool FULL>
__global__ void __launch_bounds__(WAVES * 64, 2) attention_cached_kernel(const AttentionCachedArgs a) {
  using S = Stream<DT, C8, DU, NQ, FULL>;
  constexpr int KS = S::KS, VC = S::VC, ES = S::ES, KW = S::KW, VW = S::VW, ROWS = S::ROWS, PITCH = DU + 4;
  __shared__ __attribute__((aligned(16))) float s_o[WAVES][ROWS][PITCH];
  __shared__ float s_m[WAVES][ROWS], s_l[WAVES][ROWS];

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r16 = lane & 15, g4 = lane >> 4;

  Share w;
  bool begins = true;
  if (a.workgroups == 0) {
    w.b = (int)blockIdx.x / (a.Hk * a.row_blocks);
    w.inner = (int)blockIdx.x - w.b * (a.Hk * a.row_blocks);
    w.s0 = w.first = 0;
    w.sb = w.per = w.left = steps_of(a, w.b);
  } else if (!share_of(a, lane, w)) {
    return;
  }
  int line = w.first;

  while (w.left > 0) {
    const int b = w.b, s0 = w.s0, n = min(w.sb - s0, w.left);  // steps of this problem
    const int hk = w.inner / a.row_blocks, rb = w.inner - hk * a.row_blocks;
    const int lk = keys_of(a, b), lq = queries_of(a, b);
    const int rows = a.G * lq, off = lk - lq, r_first = rb * ROWS;

    // keys in front of which the wave's steps begin: it has those with any key
    const int key0 = s0 * kCachedStep + wave * 32;
    const int end = min(lk, (s0 + n) * kCachedStep);
    const int steps = end > key0 ? (end - key0 + kCachedStep - 1) / kCachedStep : 0;

    Places at;
    Scales scales;
    f32x4 o[NQ][VC];
    float m[NQ];
    double total[NQ];
#pragma unroll
    for (int qb = 0; qb < NQ; ++qb) {
      m[qb] = -INFINITY;
      total[qb] = 0.0;
#pragma unroll
      for (int j = 0; j < VC; ++j) o[qb][j] = f32x4{0, 0, 0, 0};
    }
    // the places of the wave's steps t .. t + 31, two groups of 16 keys each
    auto locate = [&](int t) __attribute__((always_inline)) {
      bool there;
      const int page = at.locate(a, b, hk, key0 + (t + lane / 2) * kCachedStep + (lane & 1) * 16, end, there);
      const float f = C8 ? scales.load(a, hk, page, there) : 1.0f;
      if (C8 && f != 1.0f) {
#pragma unroll
        for (int qb = 0; qb < NQ; ++qb)
#pragma unroll
          for (int j = 0; j < VC; ++j) o[qb][j] *= f;
      }
      return f;
    };

    unsigned k_off[KS], v_off[4];
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const int c = (g4 * KS + s) * 8;
      k_off[s] = (unsigned)(r16 * (int)a.k.ss + (FULL || c < a.D ? c : 0) * ES);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) v_off[i] = (unsigned)((g4 * 4 + i) * (int)a.v.ss + (FULL || r16 * VC < a.D ? r16 * VC : 0) * ES);

    auto request_k = [&](int t, typename S::Keys &l) __attribute__((always_inline)) {
      const int e = (t & 31) * 2;
#pragma unroll
      for (int blk = 0; blk < 2; ++blk) {
        const unsigned char *k = at.k(e + blk);
        if constexpr (FULL) {  // a run of 8 KS columns, 16 bytes at a time
          constexpr int PER = 4 / KW;  // pieces of 8 columns in 16 bytes
#pragma unroll
          for (int s = 0; s < KS; s += PER) {
            unsigned x[4];
            load_words<4>(k, k_off[s], x);
#pragma unroll
            for (int i = 0; i < 4; ++i) l.k[blk][s + i / KW][i % KW] = x[i];
          }
        } else {
#pragma unroll
          for (int s = 0; s < KS; ++s) load_words<KW>(k, k_off[s], l.k[blk][s]);
        }
      }
    };
    auto request_v = [&](int t, typename S::Values &l) __attribute__((always_inline)) {
      const int e = (t & 31) * 2;
#pragma unroll
      for (int blk = 0; blk < 2; ++blk) {
        const unsigned char *v = at.v(e + blk);
#pragma unroll
        for (int i = 0; i < 4; ++i) load_words<VW>(v, v_off[i], l.v[blk * 4 + i]);
      }
    };
    auto tags_of = [&](int t) __attribute__((always_inline)) {
      const int e = (t & 31) * 2;
      typename S::Tags x;
      x.valid = (unsigned)(at.valid >> e) & 3u;
#pragma unroll
      for (int blk = 0; blk < 2; ++blk) {
        x.c[blk] = C8 ? of_lane(scales.c, e + blk) : a.scale_log2;
        x.lift[blk] = C8 ? of_lane(scales.lift, e + blk) : 0.0f;
      }
      return x;
    };

    typename S::Keys k_now;
    typename S::Values v_now;
    typename S::Tags tags, tags_next;
    if (steps > 0) {
      (void)locate(0);
      request_k(0, k_now);
      request_v(0, v_now);
      tags = tags_of(0);
    }

    int q_last[NQ];  // the last key that the lane's row sees
    u32x4 qf[NQ][KS];
#pragma unroll
    for (int qb = 0; qb < NQ; ++qb) {
      const int r = r_first + qb * 16 + r16, i = query_of(a, r);
      const bool there = r < rows;
      q_last[qb] = !there ? -1 : a.causal ? min(lk - 1, i + off) : lk - 1;
      const unsigned short *p =
          (const unsigned short *)a.q.p + (there ? (long long)b * a.q.sb + (long long)(hk * a.G + r - i * a.G) * a.q.sh + (long long)i * a.q.ss : 0);
#pragma unroll
      for (int s = 0; s < KS; ++s) qf[qb][s] = query_columns(a, p, there, (g4 * KS + s) * 8);
    }
    // keys that every row of the block sees, those past the last row aside (what they hold is dropped)
    int all_see = lk;
    if (a.causal && r_first < rows) all_see = min(lk, query_of(a, r_first) + off + 1);

    // Places of step t, where it is the first of 32, while the step before is not done.
    auto locate_ahead = [&](int t) __attribute__((always_inline)) {
      if ((t & 31) != 0) return;
      const float f = locate(t);
      if (C8 && f != 1.0f) {
#pragma unroll
        for (int blk = 0; blk < 2; ++blk) tags.lift[blk] = of_lane(scales.lift_before, 62 + blk);
      }
    };
    auto work = [&](int t, typename S::Keys &keys, typename S::Values &values, auto &&between) __attribute__((always_inline)) {
      const int key = key0 + t * kCachedStep;
      const bool edge = key + 32 > all_see || tags.valid != 3u;
      f32x4 z[NQ][2];
#pragma unroll
      for (int blk = 0; blk < 2; ++blk)
#pragma unroll
        for (int s = 0; s < KS; ++s) {
          u32x4 f;
          if constexpr (C8) {
            f = u32x4{widen2<DT, false>(keys.k[blk][s][0]), widen2<DT, true>(keys.k[blk][s][0]), widen2<DT, false>(keys.k[blk][s][1]), widen2<DT, true>(keys.k[blk][s][1])};
          } else {
            f = u32x4{keys.k[blk][s][0], keys.k[blk][s][1], keys.k[blk][s][2], keys.k[blk][s][3]};
          }
          if constexpr (!FULL) {  // columns from D on: the queries have zeros there, which a NaN would outlive
            if ((g4 * KS + s) * 8 >= a.D) f = u32x4{0, 0, 0, 0};
          }
#pragma unroll
          for (int qb = 0; qb < NQ; ++qb) z[qb][blk] = Mfma16<DT>::run(f, qf[qb][s], s == 0 ? f32x4{0, 0, 0, 0} : z[qb][blk]);
        }
      between();
      if (edge) {
        // a query does not see what lies behind its last key, nor a group without a page
#pragma unroll
        for (int blk = 0; blk < 2; ++blk) {
          const bool there = (tags.valid >> blk) & 1u;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int j = key + blk * 16 + g4 * 4 + i;
#pragma unroll
            for (int qb = 0; qb < NQ; ++qb) z[qb][blk][i] = !there || j > q_last[qb] ? -INFINITY : z[qb][blk][i];
            if (!there || j >= lk) {  // what has no key may hold anything
#pragma unroll
              for (int x = 0; x < VW; ++x) values.v[blk * 4 + i][x] = 0;
            }
          }
        }
      }
      u32x4 pf[NQ];
      bool moved = false;
      float alpha[NQ], back[2];
      const float(&c)[2] = tags.c, (&lift)[2] = tags.lift;
#pragma unroll
      for (int blk = 0; blk < 2; ++blk) back[blk] = C8 ? __builtin_amdgcn_exp2f(-lift[blk]) : 1.0f;
#pragma unroll
      for (int qb = 0; qb < NQ; ++qb) {
        float mx = -INFINITY;
#pragma unroll
        for (int blk = 0; blk < 2; ++blk)
          mx = fmaxf(mx, c[blk] * fmaxf(fmaxf(z[qb][blk][0], z[qb][blk][1]), fmaxf(z[qb][blk][2], z[qb][blk][3])));
        mx = groups_max_valu(mx);
        const bool mv = mx > m[qb] + (P_SHIFT<DT> + LAZY_MAX<DT>);  // (a first score above -inf always moves it)
        const float mn = mv ? mx - P_SHIFT<DT> : m[qb];
        alpha[qb] = mv ? __builtin_amdgcn_exp2f(m[qb] - mn) : 1.0f;
        m[qb] = mn;
        moved |= mv;
      }
      if (__any(moved)) {
#pragma unroll
        for (int qb = 0; qb < NQ; ++qb) {
          total[qb] *= (double)alpha[qb];
#pragma unroll
          for (int j = 0; j < VC; ++j) o[qb][j] *= alpha[qb];
        }
      }
#pragma unroll
      for (int qb = 0; qb < NQ; ++qb) {
        const float ref = m[qb] == -INFINITY ? 0.0f : m[qb];  // (nothing visible yet: exp2(-inf) = 0)
        float p[8], sum = 0.0f;
#pragma unroll
        for (int blk = 0; blk < 2; ++blk) {
          const float r = lift[blk] - ref;
          float four = 0.0f;
#pragma unroll
          for (int i = 0; i < 4; ++i) four += p[blk * 4 + i] = __builtin_amdgcn_exp2f(__builtin_fmaf(z[qb][blk][i], c[blk], r));
          sum += C8 ? four * back[blk] : four;
        }
        total[qb] += (double)sum;
        pf[qb] = u32x4{pack2<DT>(p[0], p[1]), pack2<DT>(p[2], p[3]), pack2<DT>(p[4], p[5]), pack2<DT>(p[6], p[7])};
      }
#pragma unroll
      for (int j = 0; j < VC; j += 2) {  // columns j and j + 1 of every chunk
        unsigned x[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          if constexpr (C8) x[i] = j % 4 == 0 ? widen2<DT, false>(values.v[i][j / 4]) : widen2<DT, true>(values.v[i][j / 4]);
          else x[i] = values.v[i][j / 2];
        }
        u32x4 lo, hi;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          lo[w] = __builtin_amdgcn_perm(x[2 * w + 1], x[2 * w], 0x05040100u);
          hi[w] = __builtin_amdgcn_perm(x[2 * w + 1], x[2 * w], 0x07060302u);
        }
#pragma unroll
        for (int qb = 0; qb < NQ; ++qb) {
          o[qb][j] = Mfma16<DT>::run(lo, pf[qb], o[qb][j]);
          o[qb][j + 1] = Mfma16<DT>::run(hi, pf[qb], o[qb][j + 1]);
        }
      }
    };

    // K of the next step is requested when the scores are there, V when its products are done: registers of their own for the next step's
    // loads gained nothing (8 x 8192 keys of 8 bits 27.0 us, without 26.0).
    for (int t = 0; t < steps; ++t) {
      work(t, k_now, v_now, [&]() __attribute__((always_inline)) {
        if (t + 1 >= steps) return;
        locate_ahead(t + 1);
        request_k(t + 1, k_now);
        tags_next = tags_of(t + 1);
      });
      if (t + 1 < steps) request_v(t + 1, v_now);
      tags = tags_next;
    }

    // the four waves' states meet
#pragma unroll
    for (int qb = 0; qb < NQ; ++qb) {
      const float l = groups_sum((float)total[qb]);
      if (g4 == 0) {
        s_m[wave][qb * 16 + r16] = m[qb];
        s_l[wave][qb * 16 + r16] = l;
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < VC; j += 4) {
          f32x4 x = {o[qb][j][i], o[qb][j + 1][i], o[qb][j + 2][i], o[qb][j + 3][i]};
          if constexpr (C8) x *= scales.unit();
          *(f32x4 *)&s_o[wave][qb * 16 + r16][(g4 * 4 + i) * VC + j] = x;
        }
    }
    __syncthreads();
    const bool whole = n == w.sb;
    const long long slot = 2ll * blockIdx.x + (begins ? 0 : 1);
    if (a.workgroups > 0 && s0 == 0 && threadIdx.x == 0) write_meta(a, w, line, n, begins);
#pragma unroll
    for (int qb = 0; qb < NQ; ++qb) {
      const int row = qb * 16 + (int)threadIdx.x / 16, col = (threadIdx.x & 15) * VC, r = r_first + row;
      float top = s_m[0][row];
#pragma unroll
      for (int x = 1; x < WAVES; ++x) top = fmaxf(top, s_m[x][row]);
      const float ref = top == -INFINITY ? 0.0f : top;
      float sum = 0.0f, x[VC];
#pragma unroll
      for (int j = 0; j < VC; ++j) x[j] = 0.0f;
#pragma unroll
      for (int from = 0; from < WAVES; ++from) {
        const float f = __builtin_amdgcn_exp2f(s_m[from][row] - ref);
        sum += f * s_l[from][row];
#pragma unroll
        for (int j = 0; j < VC; j += 4) {
          const f32x4 y = *(const f32x4 *)&s_o[from][row][col + j];
#pragma unroll
          for (int i = 0; i < 4; ++i) x[j + i] += f * y[i];
        }
      }
      if (r >= a.G * a.Sq) continue;
      if (!whole) {
        float *p = a.part_o + (slot * ROWS + row) * DU + col;
#pragma unroll
        for (int j = 0; j < VC; j += 4) *(f32x4 *)(p + j) = f32x4{x[j], x[j + 1], x[j + 2], x[j + 3]};
        if (col == 0) {
          a.part_ml[2 * (slot * ROWS + row)] = top;
          a.part_ml[2 * (slot * ROWS + row) + 1] = sum;
        }
        continue;
      }
      const int i = query_of(a, r), h = hk * a.G + r - i * a.G;
      const bool there = r < rows && sum != 0.0f;  // a query of the sequence that sees a key
      const float inv = sum > 0.0f ? 1.0f / sum : sum;  // (NaN stays)
      unsigned short *p = (unsigned short *)a.o.p + (long long)b * a.o.sb + (long long)h * a.o.sh + (long long)i * a.o.ss + col;
      unsigned out[VC / 2];
#pragma unroll
      for (int j = 0; j < VC; j += 2) out[j / 2] = there ? pack2<DT>(x[j] * inv, x[j + 1] * inv) : 0u;
      if (col < a.D) {
        if (a.o_vec) {
#pragma unroll
          for (int j = 0; j < VC / 2; j += 2) *(u32x2 *)(p + 2 * j) = u32x2{out[j], out[j + 1]};
        } else {
#pragma unroll
          for (int j = 0; j < VC; ++j) p[j] = (unsigned short)(out[j / 2] >> (j % 2 * 16));
        }
      }
      if (col == 0 && a.lse != nullptr)
        a.lse[(long long)b * a.lse_sb + (long long)h * a.lse_sh + (long long)i * a.lse_ss] = there ? (top + __builtin_amdgcn_logf(sum)) * LN2 : -INFINITY;
    }
    line += n;
    w.left -= n;
    if (w.left > 0) {
      __syncthreads();  // (before the next problem's states)
      begins = false;
      next_problem(a, w);
    }
  }
}

// Joins the parts of problems that were cut between workgroups.  Blocks of up to 32 rows have up to a part from every workgroup: a workgroup
// for each row of a problem, its four waves taking the parts in turn (TOGETHER).  Blocks of 128 rows have few parts and many rows: a wave
// for each.  Bound by the latency of three loads one after another, 3.9 us for 64 problems of 4 rows in 4 parts.
template <int DT, int DU, bool TOGETHER>
__global__ void __launch_bounds__(256) attention_cached_join_kernel(const AttentionCachedArgs a) {
  constexpr int C = DU / 64;
  typedef float Columns __attribute__((ext_vector_type(C)));
  __shared__ float s_o[4][DU], s_l[4];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), per_b = a.Hk * a.row_blocks;
  const int row = TOGETHER ? (int)blockIdx.x : (int)blockIdx.x * 4 + wave;
  const int s0 = a.meta[2 * blockIdx.y], parts = a.meta[2 * blockIdx.y + 1];
  const int b = (int)blockIdx.y / per_b, inner = (int)blockIdx.y - b * per_b;
  const int hk = inner / a.row_blocks, rb = inner - hk * a.row_blocks, r = rb * a.rows + row;
  if (s0 < 0 || r >= a.G * a.Sq) return;  // (not cut; a workgroup whose waves share a row leaves as a whole)
  // (nobody may have written them, where lengths were changed while they were read)
  if (parts < 1 || parts > a.all_slots || s0 + (long long)a.slots * (parts - 1) >= a.all_slots) return;
  auto at = [&](int i) { return (long long)(i == 0 ? s0 : (s0 & -a.slots) + a.slots * i) * a.rows + row; };

  float m = -INFINITY;
  for (int i = lane; i < parts; i += 64) m = fmaxf(m, a.part_ml[2 * at(i)]);
  m = wave_max(m);
  const float ref = m == -INFINITY ? 0.0f : m;
  float sum = 0.0f;
  Columns x = {};
#pragma unroll 4
  for (int i = TOGETHER ? wave : 0; i < parts; i += TOGETHER ? 4 : 1) {
    const long long p = at(i);
    const float f = __builtin_amdgcn_exp2f(a.part_ml[2 * p] - ref);
    sum += f * a.part_ml[2 * p + 1];
    x += f * *(const Columns *)(a.part_o + p * DU + lane * C);  // (columns from D on are never written, nor used)
  }
  if constexpr (TOGETHER) {
    *(Columns *)&s_o[wave][lane * C] = x;
    if (lane == 0) s_l[wave] = sum;
    __syncthreads();
    if (wave != 0) return;
    sum = (s_l[0] + s_l[1]) + (s_l[2] + s_l[3]);
    x = Columns{};
#pragma unroll
    for (int w = 0; w < 4; ++w) x += *(const Columns *)&s_o[w][lane * C];
  }
  const int i = query_of(a, r), h = hk * a.G + r - i * a.G;
  const bool there = r < a.G * queries_of(a, b) && sum != 0.0f;
  const float inv = sum > 0.0f ? 1.0f / sum : sum;  // (NaN stays)
  unsigned short *o = (unsigned short *)a.o.p + (long long)b * a.o.sb + (long long)h * a.o.sh + (long long)i * a.o.ss;
#pragma unroll
  for (int c = 0; c < C; ++c)
    if (lane * C + c < a.D) o[lane * C + c] = there ? (unsigned short)pack2<DT>(x[c] * inv, 0.0f) : (unsigned short)0;
  if (lane == 0 && a.lse != nullptr)
    a.lse[(long long)b * a.lse_sb + (long long)h * a.lse_sh + (long long)i * a.lse_ss] = there ? (m + __builtin_amdgcn_logf(sum)) * LN2 : -INFINITY;
}

template <int DT, int DU, int NQ>
void launch_rows(const AttentionCachedArgs &a, bool e4m3, hipStream_t stream) {
  const dim3 grid((unsigned)(a.workgroups > 0 ? a.workgroups : a.B * a.Hk * a.row_blocks)), block(WAVES * 64);
  const bool full = a.D == DU;
  if (e4m3 && full) hipLaunchKernelGGL((attention_cached_kernel<DT, true, DU, NQ, true>), grid, block, 0, stream, a);
  else if (e4m3) hipLaunchKernelGGL((attention_cached_kernel<DT, true, DU, NQ, false>), grid, block, 0, stream, a);
  else if (full) hipLaunchKernelGGL((attention_cached_kernel<DT, false, DU, NQ, true>), grid, block, 0, stream, a);
  else hipLaunchKernelGGL((attention_cached_kernel<DT, false, DU, NQ, false>), grid, block, 0, stream, a);
}
template <int DT, int DU>
int launch_width(const AttentionCachedArgs &a, bool e4m3, hipStream_t stream) {
  hipError_t e;
  if (a.rows > 32) {
    e = (hipError_t)launch_attention_cached_tiles(a, DT, e4m3, stream);
  } else {
    if (a.rows == 32) launch_rows<DT, DU, 2>(a, e4m3, stream);
    else launch_rows<DT, DU, 1>(a, e4m3, stream);
    e = hipGetLastError();
  }
  if (e != hipSuccess || a.meta == nullptr) return (int)e;
  const unsigned rows = (unsigned)std::min(a.G * a.Sq, a.rows), problems = (unsigned)(a.B * a.Hk * a.row_blocks);
  if (a.rows <= 32) hipLaunchKernelGGL((attention_cached_join_kernel<DT, DU, true>), dim3(rows, problems), dim3(256), 0, stream, a);
  else hipLaunchKernelGGL((attention_cached_join_kernel<DT, DU, false>), dim3((rows + 3) / 4, problems), dim3(256), 0, stream, a);
  return (int)hipGetLastError();
}

}  // namespace

int launch_attention_cached(const AttentionCachedArgs &a, int dtype, bool e4m3, hipStream_t stream) {
  if (a.D <= 64) return dtype == DT_F16 ? launch_width<DT_F16, 64>(a, e4m3, stream) : launch_width<DT_BF16, 64>(a, e4m3, stream);
  return dtype == DT_F16 ? launch_width<DT_F16, 128>(a, e4m3, stream) : launch_width<DT_BF16, 128>(a, e4m3, stream);
}

}  // namespace tracea_amd
