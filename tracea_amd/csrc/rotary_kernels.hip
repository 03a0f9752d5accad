// Rotary positions on several axes, gfx950: pair p of every head of a token is turned by the angle position[axis of p] * freq[p].
//   (u, v) -> (u cos - v sin, v cos + u sin)      inverse: the angle's other sign (the rotation's transpose, its gradient)
//
// Bound by memory: every element is read once and written once.  A thread takes 16 bytes of u and 16 bytes of v of one token
// through some heads, so that the sine and cosine of a pair, and the position behind them, are worked out once
// per group of heads instead of once per element.  Where the heads of a token lie side by side, some neighbouring threads take them in
// turn, or a wave would touch a short piece of eight tokens at a time.
// Measured: S24960 H32:8 D128 bf16 98 us = 5.2 TB/s in either layout (a large copy reaches 4.8), B8 H12:12 S1024 D64 f32 18 us = 5.6 TB/s,
// with a quarter of the columns copied 21 us; B1 H12:12 S197 f16 5.0 us, a launch.
#include "contraction_kernel.hpp"
#include "rotation.hpp"
#include "train.hpp"

namespace tracea_amd {

namespace {

template <typename T, int E>
struct alignas(sizeof(T) * E) Piece {
  T x[E];
};

template <typename T, int E, bool ADJ>
__device__ __forceinline__ void rotate(const T *in, T *out, int at_u, int at_v, const float (&c)[E], const float (&s)[E]) {
  using P = Piece<T, E>;
  const P u = *(const P *)(in + at_u), v = *(const P *)(in + at_v);
  P a, b;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    if constexpr (ADJ && E > 1) {  // pairs side by side: the first half of them in u, the second in v
      const P &w = e < E / 2 ? u : v;
      P &r = e < E / 2 ? a : b;
      const int i = 2 * (e % (E / 2));
      const float x = (float)w.x[i], y = (float)w.x[i + 1];
      r.x[i] = (T)(x * c[e] - y * s[e]);
      r.x[i + 1] = (T)(y * c[e] + x * s[e]);
    } else {
      const float x = (float)u.x[e], y = (float)v.x[e];
      a.x[e] = (T)(x * c[e] - y * s[e]);
      b.x[e] = (T)(y * c[e] + x * s[e]);
    }
  }
  *(P *)(out + at_u) = a;
  *(P *)(out + at_v) = b;
}

template <typename T, int E, bool ADJ>
__global__ void __launch_bounds__(256) rotary_kernel(const RotaryArgs a) {
  using P = Piece<T, E>;
  // pieces of a token: those with E pairs, then those of the columns that are copied
  const int turned = a.P / E, all = turned + (a.D - 2 * a.P) / E;
  int piece, slot, i;
  long long b;
  auto split = [&](auto id) __attribute__((always_inline)) {
    using N = decltype(id);
    const N row = id / (N)all, token = row / (N)a.beside, entry = token / (N)a.S;
    piece = (int)(id - row * (N)all);
    slot = (int)(row - token * (N)a.beside);
    i = (int)(token - entry * (N)a.S);
    b = (long long)entry;
  };
  if (gridDim.z == 1) split(blockIdx.x * 256u + threadIdx.x);  // (the divisions in 32 bits where they fit)
  else split(((unsigned long long)blockIdx.z * gridDim.x + blockIdx.x) * 256u + threadIdx.x);
  if (b >= a.B) return;
  const int h0 = blockIdx.y * a.heads_per_group + slot, h1 = min((int)(blockIdx.y + 1) * a.heads_per_group, a.Hq + a.Hk);
  auto heads = [&](auto &&body) __attribute__((always_inline)) {
    int h = h0;
    auto walk = [&](const HeadView &tin, const HeadView &tout, int first, int end) __attribute__((always_inline)) {
      const T *in = (const T *)tin.p + b * tin.sb + (long long)(h - first) * tin.sh + (long long)i * tin.ss;
      T *out = (T *)tout.p + b * tout.sb + (long long)(h - first) * tout.sh + (long long)i * tout.ss;
      for (; h < end; h += a.beside, in += a.beside * tin.sh, out += a.beside * tout.sh) body(in, out);
    };
    walk(a.q, a.q_out, 0, min(h1, a.Hq));
    walk(a.k, a.k_out, a.Hq, h1);
  };
  if (piece >= turned) {
    const int at = 2 * a.P + (piece - turned) * E;
    heads([&](const T *in, T *out) {
      if (in != out) *(P *)(out + at) = *(const P *)(in + at);
    });
    return;
  }
  const int at_u = ADJ ? 2 * piece * E : piece * E, at_v = ADJ ? at_u + E : at_u + a.P;
  float c[E], s[E];
  const int *pos = a.positions + b * a.pos_sb + (long long)i * a.pos_ss;
  const float sign = a.inverse ? -1.0f : 1.0f;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int p = piece * E + e;
    int axis = 0;
    for (int x = 1; x < a.axes; ++x) axis += p >= a.first[x];
    turn(pos[axis], a.inv_freq[p], sign, c[e], s[e]);
  }
  heads([&](const T *in, T *out) __attribute__((always_inline)) { rotate<T, E, ADJ>(in, out, at_u, at_v, c, s); });
}

template <typename T, int E>
int launch(const RotaryArgs &a, hipStream_t stream) {
  const long long threads = (long long)a.B * a.S * a.beside * (a.P / E + (a.D - 2 * a.P) / E);
  // (at most 2^31 threads along x: a launch of 2^32 and more drops some of them without an error)
  const long long blocks = (threads + 255) / 256, most = 1ll << 23, turns = (blocks + most - 1) / most;
  const dim3 grid((unsigned)((blocks + turns - 1) / turns), (unsigned)((a.Hq + a.Hk + a.heads_per_group - 1) / a.heads_per_group), (unsigned)turns);
  if (a.adjacent) hipLaunchKernelGGL((rotary_kernel<T, E, true>), grid, dim3(256), 0, stream, a);
  else hipLaunchKernelGGL((rotary_kernel<T, E, false>), grid, dim3(256), 0, stream, a);
  return (int)hipGetLastError();
}

}  // namespace

int launch_rotary(const RotaryArgs &a, int dtype, hipStream_t stream) {
  if (dtype == DT_F32) return a.vec ? launch<float, 4>(a, stream) : launch<float, 1>(a, stream);
  if (dtype == DT_F16) return a.vec ? launch<_Float16, 8>(a, stream) : launch<_Float16, 1>(a, stream);
  return a.vec ? launch<__bf16, 8>(a, stream) : launch<__bf16, 1>(a, stream);
}

}  // namespace tracea_amd
