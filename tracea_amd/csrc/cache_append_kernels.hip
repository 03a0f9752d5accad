// Appending keys and values to a cache in pages, gfx950: keys (and queries) are turned by their positions on the way, and in 8 bits a page and head
// has one scale.
//   16 bits  cache[page, h, place] = R x                       q' = R q
//   8 bits   need = least power of two with max|R x| <= 448 need over the new tokens of the page and head (finite ones, 2^-126 or more)
//            scale = max(old, need), old = 0 where the page begins with a new token
//            code = e4m3(R x / scale), the page's other codes e4m3(code old / scale)
// A scale that is a power of two moves codes by whole exponents: it costs no mantissa bit whatever the values are, rescaling other codes is
// exact except below the normal codes, and so a cache is the same, up to these, however its tokens were cut into calls.
//
// A workgroup has the tokens of one sequence that fall into one page, for some of the heads: no other writes that page and head, so that scales
// need no atomics across workgroups.  Sines and cosines of its tokens are kept in LDS for its heads.  Two kernels: cache_append_held_kernel where
// rows are in whole pieces of 8 and a workgroup's tokens fit its registers (256 of 128 columns), cache_append_kernel for everything else.  Few large
// pages leave few workgroups: the prompts below into pages of 512 / 2048 / 8192 tokens 194 / 748 / 1490 us, in 16 bits 116 / 440 / 871.
//
// Two prompts of 4096 tokens, 32 heads of queries and 8 of keys, 128 columns, bf16 into pages of 64 tokens in 8 bits: 52 us, 3.5 TB/s of 5.06 that
// a copy reaches, bound by the vector work beside the loads (a sine and cosine per token and pair, each operand turned twice, codes) and by a
// workgroup's chain of loads, largest value and stores; in 16 bits 50 us, 4.0 TB/s.  One token of 16 sequences: 7 us, latency only.
#include <type_traits>

#include "cache.hpp"
#include "contraction_kernel.hpp"
#include "rotation.hpp"

namespace tracea_amd {

namespace {

template <typename T, int E>
struct alignas(sizeof(T) * E) Piece {
  T x[E];
};
template <int E>
struct alignas(E) Codes {
  unsigned char x[E];
};

// The least power of two by which `largest` (finite) is at most 448 = 1.75 2^8, at least 2^-126.
__device__ __forceinline__ float scale_for(float largest) {
  const unsigned bits = __builtin_bit_cast(unsigned, largest);
  const int e = (int)(bits >> 23) - 8 + ((bits & 0x7fffffu) > 0x600000u);
  return __builtin_bit_cast(float, (unsigned)(e < 1 ? 1 : e) << 23);
}
// e4m3 codes of two values up to 448, rounded to nearest, ties to even; infinities and NaN become NaN
__device__ __forceinline__ unsigned encode2(float a, float b) { return (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false) & 0xffffu; }
template <int E>
__device__ __forceinline__ Codes<E> encode(const float (&x)[E], float inv) {
  Codes<E> c;
  if constexpr (E == 1) {
    c.x[0] = (unsigned char)encode2(x[0] * inv, 0.0f);
  } else {
#pragma unroll
    for (int e = 0; e < E; e += 2) {
      const unsigned two = encode2(x[e] * inv, x[e + 1] * inv);
      c.x[e] = (unsigned char)two;
      c.x[e + 1] = (unsigned char)(two >> 8);
    }
  }
  return c;
}

// Codes of a head of a page of PT rows but for `count` new ones from `first` on, times f (a power of two below 1), by the first threads of a
// workgroup.  (Rows behind the new ones as well: they may hold tokens, where a call writes again what a sequence had.)
__device__ __forceinline__ void rescale(unsigned char *head, long long apart, int PT, int first, int count, int D, float f, int threads) {
  for (int i = threadIdx.x; i < (PT - count) * (D / 8); i += threads) {
    int row = i / (D / 8);
    const int at = (i - row * (D / 8)) * 8;
    row += row >= first ? count : 0;
    u32x2 *p = (u32x2 *)(head + row * apart + at);
    const u32x2 x = *p;
    u32x2 y;
#pragma unroll
    for (int d = 0; d < 2; ++d) {
      const unsigned lo = encode2(__builtin_amdgcn_cvt_f32_fp8((int)x[d], 0) * f, __builtin_amdgcn_cvt_f32_fp8((int)x[d], 1) * f);
      const unsigned hi = encode2(__builtin_amdgcn_cvt_f32_fp8((int)x[d], 2) * f, __builtin_amdgcn_cvt_f32_fp8((int)x[d], 3) * f);
      y[d] = lo | hi << 16;
    }
    *p = y;
  }
}

// Any sizes, E columns at a time (8, or 4, 2 or 1 where pairs, strides or addresses do not go into that): angles of up to kAppendAngles pairs at
// once, and in 8 bits operands are read twice, for the largest value and for the codes; the second time they come from the caches.
template <typename T, bool C8, int E, bool ADJ>
__global__ void __launch_bounds__(256) cache_append_kernel(const CacheAppendArgs a) {
  __shared__ float s_cos[kAppendAngles], s_sin[kAppendAngles];
  __shared__ unsigned s_max[2][kAppendHeads];   // largest finite magnitudes, as bits
  __shared__ float s_inv[2][kAppendHeads], s_move[2][kAppendHeads];
  const int b = blockIdx.y, j = (int)blockIdx.x / a.groups, grp = (int)blockIdx.x - j * a.groups, PT = a.table.P;
  const long long start = a.starts[b] > 0 ? a.starts[b] : 0;
  const int n = a.lengths != nullptr ? min(max(a.lengths[b], 0), a.T) : a.T;
  const long long slot = (unsigned)start / (unsigned)PT + j, base = slot * PT - start;  // of the page, in new tokens
  const int lo = base > 0 ? (int)min(base, (long long)a.T) : 0, hi = (int)min(base + PT, (long long)a.T), end = min(hi, n);  // (from `end` on: queries' zeros)
  if (lo >= hi) return;
  const int h0 = min(a.Hk, grp * a.heads), h1 = min(a.Hk, h0 + a.heads), q0 = min(a.Hq, grp * a.queries), q1 = min(a.Hq, q0 + a.queries);
  const int page = page_of(a.table, b, slot);
  const bool there = page >= 0 && end > lo;
  const int heads = h1 - h0;

  const int pair_pieces = a.P / E, straight = (a.D - 2 * a.P) / E, pieces = pair_pieces + straight, all = a.D / E;
  const int chunk = append_tokens_at_once(a.P);

  auto angles = [&](int from, int to) __attribute__((always_inline)) {
    for (int i = threadIdx.x; i < (to - from) * a.P; i += 256) {
      const int t = from + i / a.P, p = i - (t - from) * a.P;
      int axis = 0;
      for (int x = 1; x < a.axes; ++x) axis += p >= a.first[x];
      const double position = a.positions != nullptr ? (double)a.positions[b * a.pos_sb + t * a.pos_ss + axis] : (double)((unsigned)start + (unsigned)t);
      float c, sn;
      turn(position, a.inv_freq[p], 1.0f, c, sn);
      s_cos[i] = c;
      s_sin[i] = sn;
    }
    __syncthreads();
  };
  // Where piece `piece` of a row lies: columns at u .. and, of a pair piece, at v .. (else v < 0)
  auto columns = [&](int piece, int &at_u, int &at_v) __attribute__((always_inline)) {
    const bool pair = piece < pair_pieces;
    at_u = !pair ? 2 * a.P + (piece - pair_pieces) * E : ADJ ? 2 * piece * E : piece * E;
    at_v = !pair ? -1 : ADJ ? at_u + E : at_u + a.P;
  };
  // Its values, turned by the angles from `angle` on.
  auto turned = [&](const T *row, int angle, int at_u, int at_v, float (&u)[E], float (&v)[E]) __attribute__((always_inline)) {
    const Piece<T, E> x = *(const Piece<T, E> *)(row + at_u), y = *(const Piece<T, E> *)(row + (at_v < 0 ? at_u : at_v));
    const bool pair = at_v >= 0;
    if (!pair) angle = 0;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      constexpr bool SIDE = ADJ && E > 1;  // the first half of the pairs in x, the second in y
      constexpr int H = E > 1 ? E / 2 : 1;
      const int i = 2 * (e % H);
      const float p = (float)(!SIDE ? x.x[e] : e < H ? x.x[i] : y.x[i]), q = (float)(!SIDE ? y.x[e] : e < H ? x.x[i + 1] : y.x[i + 1]);
      const float c = s_cos[angle + e], s = s_sin[angle + e], first = p * c - q * s, second = q * c + p * s;
      if constexpr (!SIDE) {
        u[e] = first;
        v[e] = second;
      } else if (e < H) {
        u[i] = first;
        u[i + 1] = second;
      } else {
        v[i] = first;
        v[i + 1] = second;
      }
    }
#pragma unroll
    for (int e = 0; e < E; ++e) u[e] = pair ? u[e] : (float)x.x[e];
  };
  auto store16 = [&](T *row, int at, const float (&x)[E]) __attribute__((always_inline)) {
    Piece<T, E> y;
#pragma unroll
    for (int e = 0; e < E; ++e) y.x[e] = (T)x[e];
    *(Piece<T, E> *)(row + at) = y;
  };
  auto largest = [](const float (&x)[E], float top) __attribute__((always_inline)) {
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const float y = fabsf(x[e]);
      top = y < INFINITY ? fmaxf(top, y) : top;
    }
    return top;
  };

  if (C8 && there) {
    for (int i = threadIdx.x; i < heads; i += 256) s_max[0][i] = s_max[1][i] = 0;
    for (int from = lo; from < end; from += chunk) {
      const int to = min(end, from + chunk);
      __syncthreads();
      angles(from, to);
      for (int h = 0; h < heads; ++h) {
        float k_top = 0.0f, v_top = 0.0f;
        for (int i = threadIdx.x; i < (to - from) * pieces; i += 256) {
          const int row = i / pieces, piece = i - row * pieces, t = from + row;
          int at_u, at_v;
          float u[E], v[E];
          columns(piece, at_u, at_v);
          turned((const T *)a.k.p + b * a.k.sb + (h0 + h) * a.k.sh + t * a.k.ss, row * a.P + piece * E, at_u, at_v, u, v);
          k_top = largest(u, k_top);
          if (at_v >= 0) k_top = largest(v, k_top);
        }
        for (int i = threadIdx.x; i < (to - from) * all; i += 256) {
          const int row = i / all, piece = i - row * all, t = from + row;
          const Piece<T, E> x = *(const Piece<T, E> *)((const T *)a.v.p + b * a.v.sb + (h0 + h) * a.v.sh + t * a.v.ss + piece * E);
          float u[E];
#pragma unroll
          for (int e = 0; e < E; ++e) u[e] = (float)x.x[e];
          v_top = largest(u, v_top);
        }
#pragma unroll
        for (int m = 1; m < 64; m <<= 1) {
          k_top = fmaxf(k_top, __shfl_xor(k_top, m, 64));
          v_top = fmaxf(v_top, __shfl_xor(v_top, m, 64));
        }
        if ((threadIdx.x & 63) == 0) {  // (magnitudes compare as their bits do)
          atomicMax(&s_max[0][h], __builtin_bit_cast(unsigned, k_top));
          atomicMax(&s_max[1][h], __builtin_bit_cast(unsigned, v_top));
        }
      }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < 2 * heads; i += 256) {
      const int w = i / heads, h = i - w * heads;
      float *scale = w == 0 ? a.ks.p + page * a.ks.sn + (h0 + h) * a.ks.sh : a.vs.p + page * a.vs.sn + (h0 + h) * a.vs.sh;
      const float old = base >= 0 ? 0.0f : *scale, now = fmaxf(old, scale_for(__builtin_bit_cast(float, s_max[w][h])));
      *scale = now;
      s_inv[w][h] = 1.0f / now;
      s_move[w][h] = old < now ? old / now : 1.0f;
    }
    __syncthreads();
    // the page's other codes, where the scale has grown
    const int first = (int)(lo - base);
    if (base < 0)
      for (int w = 0; w < 2; ++w)
        for (int h = 0; h < heads; ++h) {
          const float f = s_move[w][h];
          if (f == 1.0f) continue;
          if (w == 0) rescale(a.kc.p + page * a.kc.sn + (h0 + h) * a.kc.sh, a.kc.ss, PT, first, end - lo, a.D, f, 256);
          else rescale(a.vc.p + page * a.vc.sn + (h0 + h) * a.vc.sh, a.vc.ss, PT, first, end - lo, a.D, f, 256);
        }
  }

  for (int from = lo; from < hi; from += chunk) {
    const int to = min(hi, from + chunk), last = there ? min(to, end) : from;  // (keys of tokens with a place)
    __syncthreads();
    angles(from, to);
    for (int i = threadIdx.x; i < heads * (last - from) * pieces; i += 256) {
      const int row = i / pieces, piece = i - row * pieces, h = row / (last - from), t = from + row - h * (last - from);
      int at_u, at_v;
      float u[E], v[E];
      columns(piece, at_u, at_v);
      turned((const T *)a.k.p + b * a.k.sb + (h0 + h) * a.k.sh + t * a.k.ss, (t - from) * a.P + piece * E, at_u, at_v, u, v);
      unsigned char *to_row = a.kc.p + page * a.kc.sn + (h0 + h) * a.kc.sh + (t - base) * a.kc.ss;
      if constexpr (C8) {
        *(Codes<E> *)(to_row + at_u) = encode<E>(u, s_inv[0][h]);
        if (at_v >= 0) *(Codes<E> *)(to_row + at_v) = encode<E>(v, s_inv[0][h]);
      } else {
        store16((T *)to_row, at_u, u);
        if (at_v >= 0) store16((T *)to_row, at_v, v);
      }
    }
    for (int i = threadIdx.x; i < heads * (last - from) * all; i += 256) {
      const int row = i / all, piece = i - row * all, h = row / (last - from), t = from + row - h * (last - from);
      const Piece<T, E> x = *(const Piece<T, E> *)((const T *)a.v.p + b * a.v.sb + (h0 + h) * a.v.sh + t * a.v.ss + piece * E);
      unsigned char *to_row = a.vc.p + page * a.vc.sn + (h0 + h) * a.vc.sh + (t - base) * a.vc.ss;
      if constexpr (C8) {
        float u[E];
#pragma unroll
        for (int e = 0; e < E; ++e) u[e] = (float)x.x[e];
        *(Codes<E> *)(to_row + piece * E) = encode<E>(u, s_inv[1][h]);
      } else {
        *(Piece<T, E> *)((T *)to_row + piece * E) = x;
      }
    }
    for (int g0 = q0, count; g0 < q1; g0 += count) {
      count = min(q1 - g0, kAppendQueries);
      for (int i = threadIdx.x; i < count * (to - from) * pieces; i += 256) {
        const int row = i / pieces, piece = i - row * pieces, h = row / (to - from), t = from + row - h * (to - from);
        int at_u, at_v;
        float u[E], v[E];
        columns(piece, at_u, at_v);
        turned((const T *)a.q.p + b * a.q.sb + (g0 + h) * a.q.sh + t * a.q.ss, (t - from) * a.P + piece * E, at_u, at_v, u, v);
        T *out = (T *)a.q_out.p + b * a.q_out.sb + (g0 + h) * a.q_out.sh + t * a.q_out.ss;
        if (t >= n) {
#pragma unroll
          for (int e = 0; e < E; ++e) u[e] = v[e] = 0.0f;
        }
        store16(out, at_u, u);
        if (at_v >= 0) store16(out, at_v, v);
      }
    }
  }
}

// The same where a workgroup's tokens are few enough for their angles to be kept all at once and their operands in registers between the largest
// value and the codes: every byte is read once.  Rows on 16 bytes, pairs in fours.  Half of the workgroup's threads, SIDE, have the keys and values, the
// other half the queries, so that neither waits behind the other's loads.  A thread has up to HK couples of pieces of a head: with 2, keys and values
// are held together and queries by two heads, with 4 one after the other.  The smallest workgroup that holds a page is taken: measured with the prompts
// above, pages of 64 52 us (64 by cache_append_kernel), of 16 52 (78), of 128 57, of 256 57 (131).
// Pairs of halves whose number is not a multiple of 8 go by fours: two prompts of 4096 tokens of 80 columns, 40 of them turned, 36 us
// (129 one by one).
enum { HALVES, HALVES_IN_FOURS, SIDE_BY_SIDE };

template <typename T, bool C8, int PAIRING, int SIDE, int HK>
__global__ void __launch_bounds__(2 * SIDE) __attribute__((amdgpu_waves_per_eu(4))) cache_append_held_kernel(const CacheAppendArgs a) {
  constexpr int WAVES = SIDE / 64, PAIRS = SIDE * HK * 8, SETS = HK == 2 ? 2 : 1;
  constexpr bool ADJ = PAIRING == SIDE_BY_SIDE, FOURS = PAIRING == HALVES_IN_FOURS;
  typedef float f4 __attribute__((ext_vector_type(4)));
  __shared__ f4 s_cos[PAIRS / 4], s_sin[PAIRS / 4];
  __shared__ float s_max[2][2][WAVES];
  const int b = blockIdx.y, j = (int)blockIdx.x / a.groups, grp = (int)blockIdx.x - j * a.groups, PT = a.table.P;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, id = threadIdx.x & (SIDE - 1);
  const bool of_keys = __builtin_amdgcn_readfirstlane((int)threadIdx.x) < SIDE;
  const long long start = a.starts[b] > 0 ? a.starts[b] : 0;
  const int n = a.lengths != nullptr ? min(max(a.lengths[b], 0), a.T) : a.T;
  const long long slot = (unsigned)start / (unsigned)PT + j, base = slot * PT - start;  // of the page, in new tokens
  const int lo = base > 0 ? (int)min(base, (long long)a.T) : 0, hi = (int)min(base + PT, (long long)a.T), end = min(hi, n);  // (from `end` on: queries' zeros)
  if (lo >= hi) return;
  const int h0 = min(a.Hk, grp * a.heads), h1 = min(a.Hk, h0 + a.heads), q0 = min(a.Hq, grp * a.queries), q1 = min(a.Hq, q0 + a.queries);
  const int page = page_of(a.table, b, slot);
  const int tokens = page >= 0 && end > lo ? end - lo : 0;  // with a place
  const int turned_fours = a.P / 4, pieces = (a.D + 8) / 16;

  // A thread's pieces are the same in every head: token (from lo) and two times 8 columns, in two halves of 4 and 4: partners that are turned by
  // the angles from 4 angle, 4 angle + 4 on (pair), or columns that are not.  u and v begin 8 columns each (v < 0: there are none); by fours, u and v
  // the first half's, u1 and v1 the second's (u1 < 0: there are none).
  struct Couple {
    int t, u, v, u1, v1, angle;
    bool pair[2];
  };
  // (worked out where they are used, a few instructions: kept for a loop over heads they would fill the registers)
  const unsigned by_pieces = 0xffffffffu / (unsigned)pieces + 1;  // 0: divided by 1
  auto couple = [&](int s, int turned_of) __attribute__((always_inline)) {  // turned_of: how many of a token's halves are turned
    Couple p;
    unsigned i = (unsigned)id;
    asm volatile("" : "+v"(i));
    i += (unsigned)(s * SIDE);
    p.t = by_pieces == 0 ? (int)i : (int)__umulhi(i, by_pieces);
    const int piece = (int)i - p.t * pieces;
    p.pair[0] = 2 * piece < turned_of;
    p.pair[1] = 2 * piece + 1 < turned_of;
    if constexpr (FOURS) {
      auto half = [&](int i, bool pair, int &u, int &v) __attribute__((always_inline)) {
        u = pair ? 4 * i : 8 * i;
        v = pair ? u + a.P : u + 4;
      };
      half(2 * piece, p.pair[0], p.u, p.v);
      half(2 * piece + 1, p.pair[1], p.u1, p.v1);
      if (p.v1 >= a.D) p.u1 = -1;
    } else {
      p.u = ADJ || !p.pair[0] ? 16 * piece : 8 * piece;
      p.v = p.pair[0] && !ADJ ? p.u + a.P : p.u + 8 < a.D ? p.u + 8 : -1;
    }
    p.angle = p.pair[0] ? p.t * turned_fours + 2 * piece : 0;
    return p;
  };
  using X = Piece<T, 8>;
  // What a thread holds: couples of keys and of values, or of two heads' queries.
  u32x4 held[SETS * 2 * HK];
  // The compiler takes them for new values: it would keep all of them widened and turned from the largest value to the codes.
  auto anew = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < SETS * 2 * HK; ++i) asm volatile("" : "+v"(held[i]));
  };
  auto piece_of = [&](int i) { return __builtin_bit_cast(X, held[i]); };
  auto load_row = [&](const HeadView &x, int h, int count, int turned_of, auto first) __attribute__((always_inline)) {
    const char *at = (const char *)((const T *)x.p + b * x.sb + h * x.sh + lo * x.ss);
#pragma unroll
    for (int s = 0; s < HK; ++s) {
      const Couple p = couple(s, turned_of);
      if (p.t >= count) continue;
      const unsigned row = (unsigned)p.t * (unsigned)x.ss;
      if constexpr (FOURS) {
        auto four = [&](int c) { return *(const u32x2 *)(at + (row + (unsigned)c) * 2); };
        const u32x2 u = four(p.u), v = four(p.v), u1 = four(p.u1 < 0 ? p.u : p.u1), v1 = four(p.u1 < 0 ? p.v : p.v1);
        held[first() + s] = u32x4{u[0], u[1], u1[0], u1[1]};
        held[first() + HK + s] = u32x4{v[0], v[1], v1[0], v1[1]};
      } else {
        held[first() + s] = *(const u32x4 *)(at + (row + (unsigned)p.u) * 2);
        held[first() + HK + s] = *(const u32x4 *)(at + (row + (unsigned)(p.v < 0 ? p.u : p.v)) * 2);
      }
    }
  };
  auto turned = [&](const Couple &p, const X &x, const X &y, float (&u)[8], float (&v)[8]) __attribute__((always_inline)) {
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const bool pair = p.pair[half];
      const f4 c = s_cos[p.angle + half], sn = s_sin[p.angle + half];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int e = half * 4 + i;
        const float f = (float)(!ADJ ? x.x[e] : half == 0 ? x.x[2 * i] : y.x[2 * i]), g = (float)(!ADJ ? y.x[e] : half == 0 ? x.x[2 * i + 1] : y.x[2 * i + 1]);
        const float first = pair ? f * c[i] - g * sn[i] : f, second = pair ? g * c[i] + f * sn[i] : g;
        if constexpr (!ADJ) {
          u[e] = first;
          v[e] = second;
        } else if (half == 0) {
          u[2 * i] = first;
          u[2 * i + 1] = second;
        } else {
          v[2 * i] = first;
          v[2 * i + 1] = second;
        }
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  constexpr std::integral_constant<int, 0> ZERO{};
  constexpr std::integral_constant<int, 4> FOUR{};
  constexpr std::integral_constant<int, 8> EIGHT{};
  // ... of any value but NaN; a head that has an infinity is looked through again for its finite ones
  auto largest = [](const float (&x)[8], auto from, auto count, float top, bool finite) __attribute__((always_inline)) {
#pragma unroll
    for (int e = 0; e < decltype(count)::value; ++e) {
      const float y = fabsf(x[from() + e]);
      top = fmaxf(top, finite && !(y < INFINITY) ? 0.0f : y);
    }
    return top;
  };
  // ... of a couple: of what is written.  The part that is not there repeats columns that are, but as they were given: not turned where they are.
  auto largest_of = [&](const Couple &p, const float (&u)[8], const float (&v)[8], float top, bool finite) __attribute__((always_inline)) {
    if constexpr (FOURS) {
      top = largest(v, ZERO, FOUR, largest(u, ZERO, FOUR, top, finite), finite);
      const float both = largest(v, FOUR, FOUR, largest(u, FOUR, FOUR, top, finite), finite);
      return p.u1 >= 0 ? both : top;
    } else {
      top = largest(u, ZERO, EIGHT, top, finite);
      const float both = largest(v, ZERO, EIGHT, top, finite);
      return !ADJ || p.v >= 0 ? both : top;  // (a half of pairs of halves that is not there is not turned either)
    }
  };
  // A couple to a row in 16 bits or, times inv, in codes.
  auto store = [=](auto *row, const Couple &p, const float (&u)[8], const float (&v)[8], float inv) __attribute__((always_inline)) {
    constexpr bool CODES = sizeof(*row) == 1;
    auto piece = [&](int at, const float(&x)[8], auto from, auto count) __attribute__((always_inline)) {
      constexpr int N = decltype(count)::value;
      if constexpr (CODES) {
        float y[N];
#pragma unroll
        for (int e = 0; e < N; ++e) y[e] = x[from() + e];
        *(Codes<N> *)(row + at) = encode<N>(y, inv);
      } else {
        Piece<T, N> y;
#pragma unroll
        for (int e = 0; e < N; ++e) y.x[e] = (T)x[from() + e];
        *(Piece<T, N> *)(row + at) = y;
      }
    };
    if constexpr (FOURS) {
      piece(p.u, u, ZERO, FOUR);
      piece(p.v, v, ZERO, FOUR);
      if (p.u1 >= 0) {
        piece(p.u1, u, FOUR, FOUR);
        piece(p.v1, v, FOUR, FOUR);
      }
    } else {
      piece(p.u, u, ZERO, EIGHT);
      if (p.v >= 0) piece(p.v, v, ZERO, EIGHT);
    }
  };
  constexpr std::integral_constant<int, 0> FIRST{};
  constexpr std::integral_constant<int, SETS == 2 ? 2 * HK : 0> SECOND{};
  float k_old = 0.0f, v_old = 0.0f;
  auto load_head = [&](int h) __attribute__((always_inline)) {
    load_row(a.k, h, tokens, turned_fours, FIRST);
    if constexpr (SETS == 2) load_row(a.v, h, tokens, 0, SECOND);
    if (C8 && tokens > 0 && base < 0) {
      k_old = a.ks.p[page * a.ks.sn + h * a.ks.sh];
      v_old = a.vs.p[page * a.vs.sn + h * a.vs.sh];
    }
  };
  auto load_queries = [&](int h) __attribute__((always_inline)) {
    load_row(a.q, h, hi - lo, turned_fours, FIRST);
    if (SETS == 2 && h + 1 < q1) load_row(a.q, h + 1, hi - lo, turned_fours, SECOND);
  };
  // (on their way while the angles are worked out)
  if (of_keys && h0 < h1) load_head(h0);
  if (!of_keys && q0 < q1) load_queries(q0);
#pragma unroll 1
  for (int i = threadIdx.x; i < (hi - lo) * a.P; i += 2 * SIDE) {
    const int t = i / a.P, p = i - t * a.P;
    int axis = 0;
    for (int x = 1; x < a.axes; ++x) axis += p >= a.first[x];
    const double position = a.positions != nullptr ? (double)a.positions[b * a.pos_sb + (lo + t) * a.pos_ss + axis] : (double)((unsigned)start + (unsigned)(lo + t));
    float c, s;
    turn(position, a.inv_freq[p], 1.0f, c, s);
    ((float *)s_cos)[i] = c;
    ((float *)s_sin)[i] = s;
  }
  __syncthreads();

  if (!of_keys) {
    for (int h = q0; h < q1; h += SETS) {
      if (h > q0) load_queries(h);
#pragma unroll
      for (int i = 0; i < SETS; ++i) {
        if (h + i >= q1) continue;
        T *at = (T *)a.q_out.p + b * a.q_out.sb + (h + i) * a.q_out.sh + lo * a.q_out.ss;
#pragma unroll
        for (int s = 0; s < HK; ++s) {
          const Couple p = couple(s, turned_fours);
          if (p.t >= hi - lo) continue;
          float u[8], v[8];
          turned(p, piece_of(2 * HK * i + s), piece_of(2 * HK * i + HK + s), u, v);
          if (lo + p.t >= n) {
#pragma unroll
            for (int e = 0; e < 8; ++e) u[e] = v[e] = 0.0f;
          }
          store(at + (unsigned)p.t * (unsigned)a.q_out.ss, p, u, v, 1.0f);
        }
      }
    }
    if (C8 && tokens > 0)
      for (int h = h0; h < h1; ++h) {  // (those of the other half)
        __syncthreads();
        __syncthreads();
      }
    return;
  }
  // Keys or values of a head, from where they are held to their places.
  auto leave = [&](int h, const PageView &cache, const ScaleView &scales, float old, int turned_of, float (&tops)[WAVES], auto first) __attribute__((always_inline)) {
    unsigned char *head = cache.p + page * cache.sn + h * cache.sh, *rows = head + (lo - base) * cache.ss;  // of the page; of token lo in it
    float inv = 1.0f;
    if constexpr (C8) {
      float top;
      auto top_of = [&](bool finite) __attribute__((always_inline)) {
        top = 0.0f;
#pragma unroll
        for (int s = 0; s < HK; ++s) {
          const Couple p = couple(s, turned_of);
          if (p.t >= tokens) continue;
          float u[8], v[8];
          turned(p, piece_of(first() + s), piece_of(first() + HK + s), u, v);
          top = largest_of(p, u, v, top, finite);
        }
#pragma unroll
        for (int m = 1; m < 64; m <<= 1) top = fmaxf(top, __shfl_xor(top, m, 64));
      };
      top_of(false);
      if (__builtin_amdgcn_readfirstlane((int)(top == INFINITY))) {
        anew();
        top_of(true);
      }
      anew();
      if (lane == 0) tops[wave] = top;
      __syncthreads();
#pragma unroll
      for (int w = 0; w < WAVES; ++w) top = fmaxf(top, tops[w]);
      const float now = fmaxf(old, scale_for(top));
      if (threadIdx.x == 0) scales.p[page * scales.sn + h * scales.sh] = now;
      inv = 1.0f / now;
      if (base < 0 && now > old) rescale(head, cache.ss, PT, (int)(lo - base), tokens, a.D, old / now, SIDE);  // the page's other codes
    }
#pragma unroll
    for (int s = 0; s < HK; ++s) {
      const Couple p = couple(s, turned_of);
      if (p.t >= tokens) continue;
      float u[8], v[8];
      turned(p, piece_of(first() + s), piece_of(first() + HK + s), u, v);
      unsigned char *row = rows + (unsigned)p.t * (unsigned)cache.ss;
      if constexpr (C8) store(row, p, u, v, inv);
      else store((T *)row, p, u, v, 1.0f);
    }
  };
  for (int h = h0; h < h1 && tokens > 0; ++h) {
    if (h > h0) load_head(h);
    leave(h, a.kc, a.ks, k_old, turned_fours, s_max[h & 1][0], FIRST);
    if constexpr (SETS == 1) load_row(a.v, h, tokens, 0, SECOND);
    leave(h, a.vc, a.vs, v_old, 0, s_max[h & 1][1], SECOND);
  }
}

template <typename T, bool C8>
int launch(const CacheAppendArgs &a, hipStream_t stream) {
  const dim3 grid((unsigned)(a.pages * a.groups), (unsigned)a.B);
  const int tokens = a.T < a.table.P ? a.T : a.table.P, pieces = (a.D + 8) / 16;
  auto holds = [&](int side, int held) {
    return a.held && (long long)tokens * a.P <= side * held * 8 && (long long)tokens * pieces <= side * held;
  };
#define HELD(SIDE, HK)                                                                                                                     \
  if (holds(SIDE, HK)) {                                                                                                                   \
    if (a.adjacent) hipLaunchKernelGGL((cache_append_held_kernel<T, C8, SIDE_BY_SIDE, SIDE, HK>), grid, dim3(2 * SIDE), 0, stream, a);       \
    else if (a.P % 8 == 0) hipLaunchKernelGGL((cache_append_held_kernel<T, C8, HALVES, SIDE, HK>), grid, dim3(2 * SIDE), 0, stream, a);      \
    else hipLaunchKernelGGL((cache_append_held_kernel<T, C8, HALVES_IN_FOURS, SIDE, HK>), grid, dim3(2 * SIDE), 0, stream, a);               \
    return (int)hipGetLastError();                                                                                                         \
  }
  HELD(64, 2)
  HELD(128, 2)
  HELD(256, 2)
  HELD(512, 2)
  HELD(512, 4)
#undef HELD
#define PIECES(E)                                                                                                      \
  if (a.vec == E) {                                                                                                    \
    if (a.adjacent) hipLaunchKernelGGL((cache_append_kernel<T, C8, E, true>), grid, dim3(256), 0, stream, a);          \
    else hipLaunchKernelGGL((cache_append_kernel<T, C8, E, false>), grid, dim3(256), 0, stream, a);                    \
  }
  PIECES(8)
  PIECES(4)
  PIECES(2)
  PIECES(1)
#undef PIECES
  return (int)hipGetLastError();
}

}  // namespace

int launch_cache_append(const CacheAppendArgs &a, int dtype, hipStream_t stream) {
  const bool e4m3 = a.ks.p != nullptr;
  if (dtype == DT_F16) return e4m3 ? launch<_Float16, true>(a, stream) : launch<_Float16, false>(a, stream);
  return e4m3 ? launch<__bf16, true>(a, stream) : launch<__bf16, false>(a, stream);
}

}  // namespace tracea_amd
