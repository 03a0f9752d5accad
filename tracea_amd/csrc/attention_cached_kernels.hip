// Attention over a key/value cache in pages, gfx950: queries of a few rows against many keys in 16 bits, or in 8 with a scale for each page
// and head.
//
//   s_ij = scale q_i . k_j  over the keys a row sees     o_i = sum_j exp(s_ij - lse_i) v_j     lse_i = log sum_j exp(s_ij)
//   k_j = ks[page of j] code_j, v_j = vs[page of j] code_j: ks multiplies the score, vs the probability, both in fp32.
//
// Bound by reading the cache, once for all heads that share it: rows r = query G + head of the group are packed as in the attention for training.
// Nothing passes through LDS on its way: the products are v_mfma_f32_16x16x32, whose first operand is 8 values a lane, and which values these are
// is free as long as both operands agree.
//   S^T = K Q^T   of 16 keys: lane l has key l & 15 and the columns 8 KS (l >> 4) .. + 8 KS - 1, a run of the key's row; the resident
//                 queries are held by the same columns.  The result has row l & 15, keys 4 (l >> 4) + 0..3.
//   O^T += V^T P^T of 32 keys: with P as it lies, lane l's k slots are keys 4 (l >> 4) + 0..3 of both blocks of 16; it loads these 8 rows, of
//                 each the columns VC (l & 15) .. + VC - 1, and the product number j takes column j of each: a transposition by one byte
//                 permutation per two values.  The result has row l & 15 and, over the VC products, VC columns in a run for each of 4 lanes' chunks.
// Codes of 8 bits become f16 or bf16 exactly on the way (two per instruction).
//
// A wave walks every fourth block of 32 keys, the next one requested before it works on the last; a workgroup's four waves join through LDS.
// Where blocks of rows are few, all steps of 128 keys of all sequences are one line that the workgroups share out evenly, whatever the
// lengths; a problem cut between workgroups is joined by a second launch, parts in their order.
#include <type_traits>

#include "cache.hpp"
#include "contraction_kernel.hpp"

namespace tracea_amd {

namespace {

constexpr float LN2 = 0.6931471805599453f;
constexpr int WAVES = 4;

// As in the attention for training: a row's reference lies P_SHIFT powers of two below a score it has met and moves only when a step exceeds
// that score by more than LAZY_MAX.  f16 has no range below 2^-24: the shift keeps the tails of long rows.
template <int DT>
constexpr float P_SHIFT = DT == DT_F16 ? 11.0f : 0.0f;
template <int DT>
constexpr float LAZY_MAX = DT == DT_F16 ? 4.0f : 8.0f;

template <int DT>
__device__ __forceinline__ unsigned pack2(float a, float b) {
  if constexpr (DT == DT_F16) {
    typedef _Float16 half2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(unsigned, half2{(_Float16)a, (_Float16)b});
  } else {
    typedef __bf16 pair __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(unsigned, pair{(__bf16)a, (__bf16)b});
  }
}
// Two e4m3 codes of a register (its upper half: HI) in 16 bits, exactly: e4m3 has no value that f16 or bf16 lacks.
template <int DT, bool HI>
__device__ __forceinline__ unsigned widen2(unsigned codes) {
  if constexpr (DT == DT_F16) return __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)codes, 1.0f, HI));
  else return __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)codes, 1.0f, HI));
}

// max over a lane's own value and those of the other three 16-lane groups (see attention_train_kernels.hip)
__device__ __forceinline__ float groups_max(float x) {
  float a0 = x, a1 = x;
  asm volatile("s_nop 1\n\tv_permlane16_swap_b32 %0, %1" : "+v"(a0), "+v"(a1));
  float b0 = fmaxf(a0, a1), b1 = b0;
  asm volatile("s_nop 1\n\tv_permlane32_swap_b32 %0, %1" : "+v"(b0), "+v"(b1));
  return fmaxf(b0, b1);
}
__device__ __forceinline__ float groups_sum(float x) {
  x += __shfl_xor(x, 16, 64);
  return x + __shfl_xor(x, 32, 64);
}
__device__ __forceinline__ float wave_max(float x) {
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) x = fmaxf(x, __shfl_xor(x, m, 64));
  return x;
}

__device__ __forceinline__ int query_of(const AttentionCachedArgs &a, int r) {
  return a.G == 1 ? r : (int)__umulhi((unsigned)r, a.g_magic);
}
__device__ __forceinline__ int keys_of(const AttentionCachedArgs &a, int b) {
  return min(max(a.k_len[b], 0), a.table.M * a.table.P);
}
// Steps of a block of rows of sequence b: at least one, which writes what rows without keys get.
__device__ __forceinline__ int steps_of(const AttentionCachedArgs &a, int b) {
  return max(1, (keys_of(a, b) + kCachedStep - 1) / kCachedStep);
}

// Steps of all blocks of rows in front of those of sequence b (b a multiple of 64) for lane l: those in front of b + l, and of all 64 together.
__device__ __forceinline__ long long scan_steps(const AttentionCachedArgs &a, int b, int lane, long long &total, int &own) {
  own = b + lane < a.B ? steps_of(a, b + lane) : 0;
  long long x = (long long)own * (a.Hk * a.row_blocks);
  const long long mine = x;
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) {
    const long long y = __shfl_up(x, m, 64);
    if (lane >= m) x += y;
  }
  total = __shfl(x, 63, 64);
  return x - mine;
}
__device__ __forceinline__ long long uniform(long long x) {
  return (long long)(unsigned)__builtin_amdgcn_readfirstlane((int)x) | (long long)__builtin_amdgcn_readfirstlane((int)(x >> 32)) << 32;
}
// Steps of a workgroup where all of them are shared out.
__device__ __forceinline__ long long share_of(const AttentionCachedArgs &a, int lane, long long &all) {
  all = 0;
  for (int b = 0; b < a.B; b += 64) {
    long long total;
    int own;
    (void)scan_steps(a, b, lane, total, own);
    all += total;
  }
  all = uniform(all);
  const long long per = (all + a.workgroups - 1) / a.workgroups;
  return per < a.least ? a.least : per;
}

template <int DT, bool C8, int DU, int NQ, bool FULL>
struct Stream {
  static constexpr int KS = DU / 32, VC = DU / 16, ES = C8 ? 1 : 2, ROWS = 16 * NQ;
  static constexpr int KW = 2 * ES, VW = VC * ES / 4;  // registers of 8 columns of a key, of a chunk of a row of values

  // What a step loads: 32 keys.
  struct Loads {
    unsigned k[2][KS][KW];
    unsigned v[8][VW];
    float ks[2], vs[2];
    unsigned valid;  // of the two groups of 16
  };
  // Where the wave's next groups of 16 keys lie, one per lane.
  struct Places {
    unsigned k_lo, k_hi, v_lo, v_hi;
    float ks, vs;
    unsigned long long valid;
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
// (two waves a SIMD, but for the form whose loads in flight and sums fill more than half of the registers)
__global__ void __launch_bounds__(WAVES * 64, NQ == 2 && !C8 && DU == 128 ? 1 : 2) attention_cached_kernel(const AttentionCachedArgs a) {
  using S = Stream<DT, C8, DU, NQ, FULL>;
  constexpr int KS = S::KS, VC = S::VC, ES = S::ES, KW = S::KW, VW = S::VW, ROWS = S::ROWS, PITCH = DU + 4;
  __shared__ __attribute__((aligned(16))) float s_o[WAVES][ROWS][PITCH];
  __shared__ float s_m[WAVES][ROWS], s_l[WAVES][ROWS];

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r16 = lane & 15, g4 = lane >> 4;
  const int per_b = a.Hk * a.row_blocks;

  // the workgroup's share: `left` steps from step s0 of problem `inner` of sequence b
  int b, inner, s0, sb;
  long long left;
  bool fresh_start = true;
  if (a.workgroups == 0) {
    b = (int)blockIdx.x / per_b;
    inner = (int)blockIdx.x - b * per_b;
    s0 = 0;
    sb = steps_of(a, b);
    left = sb;
  } else {
    long long all;
    const long long per = share_of(a, lane, all), first = (long long)blockIdx.x * per;
    if (first >= all) return;
    left = min(per, all - first);
    long long before = 0;
    b = 0;
    for (int b0 = 0;; b0 += 64) {
      long long total;
      int own;
      const long long mine = scan_steps(a, b0, lane, total, own);
      if (uniform(before + total) > first) {
        const unsigned long long here = __ballot(before + mine <= first && own > 0);
        const int at = 63 - __clzll(here);
        b = b0 + at;
        sb = __builtin_amdgcn_readlane(own, at);
        const long long u = first - (before + uniform(__shfl(mine, at, 64)));
        inner = (int)(u / sb);
        s0 = (int)(u - (long long)inner * sb);
        break;
      }
      before += total;
    }
    b = __builtin_amdgcn_readfirstlane(b);
    inner = __builtin_amdgcn_readfirstlane(inner);
    s0 = __builtin_amdgcn_readfirstlane(s0);
    left = uniform(left);
  }

  while (left > 0) {
    const int n = (int)min((long long)(sb - s0), left);  // steps of this problem
    const int hk = inner / a.row_blocks, rb = inner - hk * a.row_blocks;
    const int lk = keys_of(a, b), lq = a.q_len != nullptr ? min(max(a.q_len[b], 0), a.Sq) : a.Sq;
    const int rows = a.G * lq, off = lk - lq, r_first = rb * ROWS;

    const unsigned char *k_head = a.k.p + hk * a.k.sh, *v_head = a.v.p + hk * a.v.sh;
    const float *ks_head = C8 ? a.ks.p + hk * a.ks.sh : nullptr, *vs_head = C8 ? a.vs.p + hk * a.vs.sh : nullptr;

    // keys in front of which the wave's steps begin: it has those with any key
    const int key0 = s0 * kCachedStep + wave * 32;
    const int end = min(lk, (s0 + n) * kCachedStep);
    const int steps = end > key0 ? (end - key0 + kCachedStep - 1) / kCachedStep : 0;

    typename S::Places at;
    float v_ref = 0.0f;  // the largest scale of values met
    float v_inv = 1.0f;
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
      const int key = key0 + (t + lane / 2) * kCachedStep + (lane & 1) * 16, group = key >> 4;
      const int slot_page = a.page_magic == 0 ? group : (int)__umulhi((unsigned)group, a.page_magic);
      int page = key < end ? page_of(a.table, b, slot_page) : -1;
      const bool there = page >= 0;
      const int place = there ? key - slot_page * a.table.P : 0;
      page = there ? page : 0;  // (something to load)
      const unsigned long long k = (unsigned long long)(k_head + page * a.k.sn + place * a.k.ss);
      const unsigned long long v = (unsigned long long)(v_head + page * a.v.sn + place * a.v.ss);
      at.k_lo = (unsigned)k; at.k_hi = (unsigned)(k >> 32);
      at.v_lo = (unsigned)v; at.v_hi = (unsigned)(v >> 32);
      at.valid = __ballot(there);
      if constexpr (C8) {
        at.ks = ks_head[page * a.ks.sn];
        at.vs = vs_head[page * a.vs.sn];
        const float top = wave_max(there ? fabsf(at.vs) : 0.0f);
        if (top > v_ref) {
          const float f = v_ref / top;
          v_ref = top;
          v_inv = 1.0f / fmaxf(v_ref, 1.17549435e-38f);
#pragma unroll
          for (int qb = 0; qb < NQ; ++qb)
#pragma unroll
            for (int j = 0; j < VC; ++j) o[qb][j] *= f;
        }
      }
    };

    unsigned k_off[KS], v_off[4];
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const int c = (g4 * KS + s) * 8;
      k_off[s] = (unsigned)(r16 * (int)a.k.ss + (FULL || c < a.D ? c : 0) * ES);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) v_off[i] = (unsigned)((g4 * 4 + i) * (int)a.v.ss + (FULL || r16 * VC < a.D ? r16 * VC : 0) * ES);

    auto request = [&](int t, typename S::Loads &l) __attribute__((always_inline)) {
      const int e = (t & 31) * 2;
      l.valid = (unsigned)(at.valid >> e) & 3u;
#pragma unroll
      for (int blk = 0; blk < 2; ++blk) {
        const unsigned char *k = (const unsigned char *)((unsigned long long)(unsigned)__builtin_amdgcn_readlane((int)at.k_lo, e + blk) |
                                                         (unsigned long long)(unsigned)__builtin_amdgcn_readlane((int)at.k_hi, e + blk) << 32);
        const unsigned char *v = (const unsigned char *)((unsigned long long)(unsigned)__builtin_amdgcn_readlane((int)at.v_lo, e + blk) |
                                                         (unsigned long long)(unsigned)__builtin_amdgcn_readlane((int)at.v_hi, e + blk) << 32);
        if constexpr (FULL) {  // a run of 8 KS columns, 16 bytes at a time
          constexpr int PER = 4 / KW;  // pieces of 8 columns in 16 bytes
#pragma unroll
          for (int s = 0; s < KS; s += PER) {
            unsigned w[4];
            load_words<4>(k, k_off[s], w);
#pragma unroll
            for (int i = 0; i < 4; ++i) l.k[blk][s + i / KW][i % KW] = w[i];
          }
        } else {
#pragma unroll
          for (int s = 0; s < KS; ++s) load_words<KW>(k, k_off[s], l.k[blk][s]);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) load_words<VW>(v, v_off[i], l.v[blk * 4 + i]);
        if constexpr (C8) {
          l.ks[blk] = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, at.ks), e + blk));
          l.vs[blk] = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, at.vs), e + blk));
        }
      }
    };

    typename S::Loads now, next;
    if (steps > 0) {
      locate(0);
      request(0, now);
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
      for (int s = 0; s < KS; ++s) {
        const int c = (g4 * KS + s) * 8;
        qf[qb][s] = u32x4{0, 0, 0, 0};
        if (there && c < a.D) {
          if (a.q_vec) {
            qf[qb][s] = *(const u32x4 *)(p + c);
          } else {
#pragma unroll
            for (int w = 0; w < 4; ++w) qf[qb][s][w] = (unsigned)p[c + 2 * w] | (unsigned)p[c + 2 * w + 1] << 16;
          }
        }
        if (a.negate) qf[qb][s] ^= 0x80008000u;
      }
    }
    // keys that every row of the block sees, those past the last row aside (what they hold is dropped)
    int all_see = lk;
    if (a.causal && r_first < rows) all_see = min(lk, query_of(a, r_first) + off + 1);

    auto work = [&](int t, typename S::Loads &l) __attribute__((always_inline)) {
      const int key = key0 + t * kCachedStep;
      const bool edge = key + 32 > all_see || l.valid != 3u;
      f32x4 z[NQ][2];
#pragma unroll
      for (int blk = 0; blk < 2; ++blk)
#pragma unroll
        for (int s = 0; s < KS; ++s) {
          u32x4 f;
          if constexpr (C8) {
            f = u32x4{widen2<DT, false>(l.k[blk][s][0]), widen2<DT, true>(l.k[blk][s][0]), widen2<DT, false>(l.k[blk][s][1]), widen2<DT, true>(l.k[blk][s][1])};
          } else {
            f = u32x4{l.k[blk][s][0], l.k[blk][s][1], l.k[blk][s][2], l.k[blk][s][3]};
          }
          if constexpr (!FULL) {  // columns from D on: the queries have zeros there, which a NaN would outlive
            if ((g4 * KS + s) * 8 >= a.D) f = u32x4{0, 0, 0, 0};
          }
#pragma unroll
          for (int qb = 0; qb < NQ; ++qb) z[qb][blk] = Mfma16<DT>::run(f, qf[qb][s], s == 0 ? f32x4{0, 0, 0, 0} : z[qb][blk]);
        }
      if (edge) {
        // a query does not see what lies behind its last key, nor a group without a page
#pragma unroll
        for (int blk = 0; blk < 2; ++blk) {
          const bool there = (l.valid >> blk) & 1u;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int j = key + blk * 16 + g4 * 4 + i;
#pragma unroll
            for (int qb = 0; qb < NQ; ++qb) z[qb][blk][i] = !there || j > q_last[qb] ? -INFINITY : z[qb][blk][i];
            if (!there || j >= lk) {  // what has no key may hold anything
#pragma unroll
              for (int w = 0; w < VW; ++w) l.v[blk * 4 + i][w] = 0;
            }
          }
        }
      }
      u32x4 pf[NQ];
      bool moved = false;
      float alpha[NQ], c[2], ratio[2];
#pragma unroll
      for (int blk = 0; blk < 2; ++blk) {
        c[blk] = C8 ? a.scale_log2 * l.ks[blk] : a.scale_log2;
        ratio[blk] = C8 ? l.vs[blk] * v_inv : 1.0f;
      }
#pragma unroll
      for (int qb = 0; qb < NQ; ++qb) {
        float mx = -INFINITY;
#pragma unroll
        for (int blk = 0; blk < 2; ++blk)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            if constexpr (C8) {
              // (-inf stays what it is whatever the scale)
              z[qb][blk][i] = z[qb][blk][i] == -INFINITY ? -INFINITY : z[qb][blk][i] * c[blk];
            } else {
              z[qb][blk][i] *= c[blk];
            }
            mx = fmaxf(mx, z[qb][blk][i]);
          }
        mx = groups_max(mx);
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
        for (int i = 0; i < 8; ++i) {
          p[i] = __builtin_amdgcn_exp2f(z[qb][i / 4][i % 4] - ref);
          sum += p[i];
          if constexpr (C8) p[i] *= ratio[i / 4];
        }
        total[qb] += (double)sum;
        pf[qb] = u32x4{pack2<DT>(p[0], p[1]), pack2<DT>(p[2], p[3]), pack2<DT>(p[4], p[5]), pack2<DT>(p[6], p[7])};
      }
#pragma unroll
      for (int j = 0; j < VC; j += 2) {  // columns j and j + 1 of every chunk
        unsigned x[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          if constexpr (C8) x[i] = j % 4 == 0 ? widen2<DT, false>(l.v[i][j / 4]) : widen2<DT, true>(l.v[i][j / 4]);
          else x[i] = l.v[i][j / 2];
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

    auto ahead = [&](int t, typename S::Loads &l) __attribute__((always_inline)) {
      if (t >= steps) return;
      if ((t & 31) == 0) locate(t);
      request(t, l);
    };
    for (int t = 0; t < steps; t += 2) {
      ahead(t + 1, next);
      work(t, now);
      if (t + 1 >= steps) break;
      ahead(t + 2, now);
      work(t + 1, next);
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
          if constexpr (C8) x *= fmaxf(v_ref, 1.17549435e-38f);
          *(f32x4 *)&s_o[wave][qb * 16 + r16][(g4 * 4 + i) * VC + j] = x;
        }
    }
    __syncthreads();
    const bool whole = n == sb;
    const long long slot = 2ll * blockIdx.x + (fresh_start ? 0 : 1);
#pragma unroll
    for (int qb = 0; qb < NQ; ++qb) {
      const int row = qb * 16 + (int)threadIdx.x / 16, col = (threadIdx.x & 15) * VC, r = r_first + row;
      float top = s_m[0][row];
#pragma unroll
      for (int w = 1; w < WAVES; ++w) top = fmaxf(top, s_m[w][row]);
      const float ref = top == -INFINITY ? 0.0f : top;
      float sum = 0.0f, x[VC];
#pragma unroll
      for (int j = 0; j < VC; ++j) x[j] = 0.0f;
#pragma unroll
      for (int w = 0; w < WAVES; ++w) {
        const float f = __builtin_amdgcn_exp2f(s_m[w][row] - ref);
        sum += f * s_l[w][row];
#pragma unroll
        for (int j = 0; j < VC; j += 4) {
          const f32x4 y = *(const f32x4 *)&s_o[w][row][col + j];
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
    left -= n;
    if (left > 0) {
      __syncthreads();  // (before the next problem's states)
      fresh_start = false;
      s0 = 0;
      if (++inner == per_b) {
        inner = 0;
        ++b;
        sb = steps_of(a, b);
      }
    }
  }
}

// Joins the parts of problems that were cut between workgroups: a workgroup for each row of a problem, its four waves
// taking the parts in turn.
template <int DT, int DU, int NQ>
__global__ void __launch_bounds__(256) attention_cached_join_kernel(const AttentionCachedArgs a) {
  constexpr int ROWS = 16 * NQ, C = DU / 64;
  __shared__ float s_o[4][DU], s_l[4];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, per_b = a.Hk * a.row_blocks;
  const int b = (int)blockIdx.y / per_b, inner = (int)blockIdx.y - b * per_b, row = blockIdx.x;
  const int hk = inner / a.row_blocks, rb = inner - hk * a.row_blocks, r = rb * ROWS + row;
  if (r >= a.G * a.Sq) return;
  long long all, before = 0;
  const long long per = share_of(a, lane, all);
  int sb = 0;
  for (int b0 = 0; b0 <= b; b0 += 64) {
    long long total;
    int own;
    const long long mine = scan_steps(a, b0, lane, total, own);
    if (b < b0 + 64) {
      before += __shfl(mine, b - b0, 64);
      sb = __shfl(own, b - b0, 64);
    } else {
      before += total;
    }
  }
  const long long first = uniform(before) + (long long)inner * sb, last = first + sb - 1;
  const long long w0 = first / per, w1 = last / per;
  if (w0 == w1) return;  // (not cut)
  auto slot_of = [&](long long w) { return 2 * w + (w == w0 && w0 * per != first ? 1 : 0); };  // (a workgroup's second part begins behind its start)

  float m = -INFINITY;
  for (long long w = w0 + lane; w <= w1; w += 64) m = fmaxf(m, a.part_ml[2 * (slot_of(w) * ROWS + row)]);
  m = wave_max(m);
  const float ref = m == -INFINITY ? 0.0f : m;
  float sum = 0.0f, x[C];
#pragma unroll
  for (int c = 0; c < C; ++c) x[c] = 0.0f;
#pragma unroll 4
  for (long long w = w0 + wave; w <= w1; w += 4) {
    const long long at = slot_of(w) * ROWS + row;
    const float f = __builtin_amdgcn_exp2f(a.part_ml[2 * at] - ref);
    sum += f * a.part_ml[2 * at + 1];
#pragma unroll
    for (int c = 0; c < C; ++c) x[c] += f * a.part_o[at * DU + lane * C + c];
  }
#pragma unroll
  for (int c = 0; c < C; ++c) s_o[wave][lane * C + c] = x[c];
  if (lane == 0) s_l[wave] = sum;
  __syncthreads();
  const int col = threadIdx.x;
  if (col >= a.D) return;
  sum = (s_l[0] + s_l[1]) + (s_l[2] + s_l[3]);
  const int i = query_of(a, r), h = hk * a.G + r - i * a.G;
  const int lq = a.q_len != nullptr ? min(max(a.q_len[b], 0), a.Sq) : a.Sq;
  const bool there = r < a.G * lq && sum != 0.0f;
  const float inv = sum > 0.0f ? 1.0f / sum : sum;
  const float y = there ? ((s_o[0][col] + s_o[1][col]) + (s_o[2][col] + s_o[3][col])) * inv : 0.0f;
  ((unsigned short *)a.o.p)[(long long)b * a.o.sb + (long long)h * a.o.sh + (long long)i * a.o.ss + col] = (unsigned short)pack2<DT>(y, 0.0f);
  if (col == 0 && a.lse != nullptr)
    a.lse[(long long)b * a.lse_sb + (long long)h * a.lse_sh + (long long)i * a.lse_ss] = there ? (m + __builtin_amdgcn_logf(sum)) * LN2 : -INFINITY;
}

template <int DT, int DU, int NQ>
int launch_rows(const AttentionCachedArgs &a, bool e4m3, hipStream_t stream) {
  const int problems = a.B * a.Hk * a.row_blocks;
  const dim3 grid((unsigned)(a.workgroups > 0 ? a.workgroups : problems)), block(WAVES * 64);
  const bool full = a.D == DU;
  if (e4m3 && full) hipLaunchKernelGGL((attention_cached_kernel<DT, true, DU, NQ, true>), grid, block, 0, stream, a);
  else if (e4m3) hipLaunchKernelGGL((attention_cached_kernel<DT, true, DU, NQ, false>), grid, block, 0, stream, a);
  else if (full) hipLaunchKernelGGL((attention_cached_kernel<DT, false, DU, NQ, true>), grid, block, 0, stream, a);
  else hipLaunchKernelGGL((attention_cached_kernel<DT, false, DU, NQ, false>), grid, block, 0, stream, a);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || a.workgroups == 0) return (int)e;
  const int rows = a.G * a.Sq < 16 * NQ ? a.G * a.Sq : 16 * NQ;
  hipLaunchKernelGGL((attention_cached_join_kernel<DT, DU, NQ>), dim3((unsigned)rows, (unsigned)problems), dim3(256), 0, stream, a);
  return (int)hipGetLastError();
}
template <int DT>
int launch_type(const AttentionCachedArgs &a, bool e4m3, hipStream_t stream) {
  if (a.D <= 64) return a.two ? launch_rows<DT, 64, 2>(a, e4m3, stream) : launch_rows<DT, 64, 1>(a, e4m3, stream);
  return a.two ? launch_rows<DT, 128, 2>(a, e4m3, stream) : launch_rows<DT, 128, 1>(a, e4m3, stream);
}

}  // namespace

int launch_attention_cached(const AttentionCachedArgs &a, int dtype, bool e4m3, hipStream_t stream) {
  return dtype == DT_F16 ? launch_type<DT_F16>(a, e4m3, stream) : launch_type<DT_BF16>(a, e4m3, stream);
}

}  // namespace tracea_amd
