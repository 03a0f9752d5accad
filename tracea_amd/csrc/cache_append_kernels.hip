// Appending keys and values to a cache in pages, gfx950: keys (and queries) are turned by their positions on the way, and in 8 bits a page and head
// has one scale.
//   16 bits  cache[page, h, place] = R x                       q' = R q
//   8 bits   need = least power of two with max|R x| <= 448 need over the new tokens of the page and head (finite ones, 2^-126 or more)
//            scale = max(old, need), old = 0 where the page begins with a new token
//            code = e4m3(R x / scale), older codes e4m3(code old / scale)
// A scale that is a power of two moves codes by whole exponents: it costs no mantissa bit whatever the values are, rescaling older codes is
// exact except below the normal codes, and so a cache is the same, up to these, however its tokens were cut into calls.
//
// A workgroup has the tokens of one sequence that fall into one page, for some of the heads: no other writes that page and head, so that scales
// need no atomics across workgroups.  Sines and cosines of its tokens are kept in LDS for its heads.  In 8 bits it reads its
// operands twice, for the largest value and for the codes; the second time they come from the caches.
#include "cache.hpp"
#include "contraction_kernel.hpp"
#include "rotation.hpp"

namespace tracea_amd {

namespace {

constexpr int ANGLES = 4096;  // pairs whose sine and cosine are kept, 32 KB

template <typename T, int E>
struct alignas(sizeof(T) * E) Piece {
  T x[E];
};
template <int E>
struct alignas(E) Codes {
  unsigned char x[E];
};

__device__ __forceinline__ float coded(float x, float inv) {  // an infinity becomes NaN: e4m3 has none
  return __builtin_isfinite(x) ? x * inv : __builtin_nanf("");
}
// The least power of two by which `largest` (finite) is at most 448 = 1.75 2^8, at least 2^-126.
__device__ __forceinline__ float scale_for(float largest) {
  const unsigned bits = __builtin_bit_cast(unsigned, largest);
  const int e = (int)(bits >> 23) - 8 + ((bits & 0x7fffffu) > 0x600000u);
  return __builtin_bit_cast(float, (unsigned)(e < 1 ? 1 : e) << 23);
}
// e4m3 codes of two values up to 448, rounded to nearest, ties to even
__device__ __forceinline__ unsigned encode2(float a, float b) { return (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false) & 0xffffu; }
template <int E>
__device__ __forceinline__ Codes<E> encode(const float (&x)[E], float inv) {
  Codes<E> c;
  if constexpr (E == 1) {
    c.x[0] = (unsigned char)encode2(coded(x[0], inv), 0.0f);
  } else {
#pragma unroll
    for (int e = 0; e < E; e += 2) {
      const unsigned two = encode2(coded(x[e], inv), coded(x[e + 1], inv));
      c.x[e] = (unsigned char)two;
      c.x[e + 1] = (unsigned char)(two >> 8);
    }
  }
  return c;
}

template <typename T, bool C8, int E, bool ADJ>
__global__ void __launch_bounds__(256) cache_append_kernel(const CacheAppendArgs a) {
  __shared__ float s_cos[ANGLES], s_sin[ANGLES];
  __shared__ unsigned s_max[2][kAppendHeads];   // largest finite magnitudes, as bits
  __shared__ float s_inv[2][kAppendHeads], s_move[2][kAppendHeads];
  const int b = blockIdx.y, j = (int)blockIdx.x / a.groups, grp = (int)blockIdx.x - j * a.groups, PT = a.table.P;
  const long long start = a.starts[b] > 0 ? a.starts[b] : 0;
  const int n = a.lengths != nullptr ? min(max(a.lengths[b], 0), a.T) : a.T;
  const long long slot = start / PT + j, base = slot * PT - start;  // of the page, in new tokens
  const int lo = base > 0 ? (int)min(base, (long long)a.T) : 0, hi = (int)min(base + PT, (long long)a.T), end = min(hi, n);  // (from `end` on: queries' zeros)
  if (lo >= hi) return;
  const int h0 = (int)((long long)a.Hk * grp / a.groups), h1 = (int)((long long)a.Hk * (grp + 1) / a.groups);
  const int q0 = (int)((long long)a.Hq * grp / a.groups), q1 = (int)((long long)a.Hq * (grp + 1) / a.groups);
  const int page = page_of(a.table, b, slot);
  const bool there = page >= 0 && end > lo;
  const int heads = h1 - h0;

  const int pair_pieces = a.P / E, straight = (a.D - 2 * a.P) / E, pieces = pair_pieces + straight, all = a.D / E;
  const int chunk = a.P > 0 ? max(1, ANGLES / a.P) : PT;

  auto angles = [&](int from, int to) __attribute__((always_inline)) {
    for (int i = threadIdx.x; i < (to - from) * a.P; i += 256) {
      const int t = from + i / a.P, p = i - (t - from) * a.P;
      int axis = 0;
      for (int x = 1; x < a.axes; ++x) axis += p >= a.first[x];
      const int position = a.positions != nullptr ? a.positions[b * a.pos_sb + t * a.pos_ss + axis] : (int)(start + t);
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
      for (int i = threadIdx.x; i < heads * (to - from) * pieces; i += 256) {
        const int row = i / pieces, piece = i - row * pieces, h = row / (to - from), t = from + row - h * (to - from);
        int at_u, at_v;
        float u[E], v[E];
        columns(piece, at_u, at_v);
      turned((const T *)a.k.p + b * a.k.sb + (h0 + h) * a.k.sh + t * a.k.ss, (t - from) * a.P + piece * E, at_u, at_v, u, v);
        float top = largest(u, 0.0f);
        if (at_v >= 0) top = largest(v, top);
        atomicMax(&s_max[0][h], __builtin_bit_cast(unsigned, top));
      }
      for (int i = threadIdx.x; i < heads * (to - from) * all; i += 256) {
        const int row = i / all, piece = i - row * all, h = row / (to - from), t = from + row - h * (to - from);
        const Piece<T, E> x = *(const Piece<T, E> *)((const T *)a.v.p + b * a.v.sb + (h0 + h) * a.v.sh + t * a.v.ss + piece * E);
        float u[E];
#pragma unroll
        for (int e = 0; e < E; ++e) u[e] = (float)x.x[e];
        atomicMax(&s_max[1][h], __builtin_bit_cast(unsigned, largest(u, 0.0f)));
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
    // older codes of the page, where the scale has grown
    const int older = base < 0 ? (int)-base : 0;
    if (older > 0)
      for (int w = 0; w < 2; ++w)
        for (int h = 0; h < heads; ++h) {
          const float f = s_move[w][h];
          if (f == 1.0f) continue;
          unsigned char *rows = w == 0 ? a.kc.p + page * a.kc.sn + (h0 + h) * a.kc.sh : a.vc.p + page * a.vc.sn + (h0 + h) * a.vc.sh;
          const long long apart = w == 0 ? a.kc.ss : a.vc.ss;
          for (int i = threadIdx.x; i < older * (a.D / 8); i += 256) {
            const int row = i / (a.D / 8), at = (i - row * (a.D / 8)) * 8;
            u32x2 *p = (u32x2 *)(rows + row * apart + at);
            const u32x2 x = *p;
            u32x2 y;
#pragma unroll
            for (int d = 0; d < 2; ++d) {
              const unsigned lo2 = encode2(__builtin_amdgcn_cvt_f32_fp8((int)x[d], 0) * f, __builtin_amdgcn_cvt_f32_fp8((int)x[d], 1) * f);
              const unsigned hi2 = encode2(__builtin_amdgcn_cvt_f32_fp8((int)x[d], 2) * f, __builtin_amdgcn_cvt_f32_fp8((int)x[d], 3) * f);
              y[d] = lo2 | hi2 << 16;
            }
            *p = y;
          }
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
    for (int i = threadIdx.x; i < (q1 - q0) * (to - from) * pieces; i += 256) {
      const int row = i / pieces, piece = i - row * pieces, h = row / (to - from), t = from + row - h * (to - from);
      int at_u, at_v;
      float u[E], v[E];
      columns(piece, at_u, at_v);
      turned((const T *)a.q.p + b * a.q.sb + (q0 + h) * a.q.sh + t * a.q.ss, (t - from) * a.P + piece * E, at_u, at_v, u, v);
      T *out = (T *)a.q_out.p + b * a.q_out.sb + (q0 + h) * a.q_out.sh + t * a.q_out.ss;
      if (t >= n) {
#pragma unroll
        for (int e = 0; e < E; ++e) u[e] = v[e] = 0.0f;
      }
      store16(out, at_u, u);
      if (at_v >= 0) store16(out, at_v, v);
    }
  }
}

template <typename T, bool C8>
int launch(const CacheAppendArgs &a, hipStream_t stream) {
  const dim3 grid((unsigned)(a.pages * a.groups), (unsigned)a.B);
  if (a.vec && a.adjacent) hipLaunchKernelGGL((cache_append_kernel<T, C8, 8, true>), grid, dim3(256), 0, stream, a);
  else if (a.vec) hipLaunchKernelGGL((cache_append_kernel<T, C8, 8, false>), grid, dim3(256), 0, stream, a);
  else if (a.adjacent) hipLaunchKernelGGL((cache_append_kernel<T, C8, 1, true>), grid, dim3(256), 0, stream, a);
  else hipLaunchKernelGGL((cache_append_kernel<T, C8, 1, false>), grid, dim3(256), 0, stream, a);
  return (int)hipGetLastError();
}

}  // namespace

int launch_cache_append(const CacheAppendArgs &a, int dtype, hipStream_t stream) {
  const bool e4m3 = a.ks.p != nullptr;
  if (dtype == DT_F16) return e4m3 ? launch<_Float16, true>(a, stream) : launch<_Float16, false>(a, stream);
  return e4m3 ? launch<__bf16, true>(a, stream) : launch<__bf16, false>(a, stream);
}

}  // namespace tracea_amd
