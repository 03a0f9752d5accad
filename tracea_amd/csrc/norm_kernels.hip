// The sum between two blocks with a norm on either side, gfx950, and its backward pass.
//   forward   n = h r1 w_post, x' = c x + gate n, y = x' r2 w_pre          r = rsqrt(mean of squares + eps)
//   backward  x^ = x' r2, g = dy w_pre, dt = dx' + r2 (g - x^ mean(g x^)), dx = c dt
//             h^ = h r1, a = dt gate w_post, dh = r1 (a - h^ mean(a h^))
//             A_b = sum over b's rows of dt h^: dgate_b = A_b w_post, dw_post = sum_b gate_b A_b; dw_pre = sum dy x^
//
// Bound by memory: one pass, each row read once and written once.  A row is held in registers by the threads of a
// workgroup (up to 256 channels: by some lanes of a wave), 8 channels each; a workgroup takes a run of rows of one batch entry,
// the next one requested ahead, with the weights and, backward, the column sums in registers all along.  The backward pass needs
// six sums over a row; all are linear in what is loaded, so that they are taken in one go and the threads meet once per row.
// Column sums leave as one partial row per workgroup and a second kernel adds these up in their order: no atomics.
// Measured (GPU time of a call, several cards; a large copy reaches 4.8 TB/s): forward C2048 T24960 bf16 89-92 us = 4.5 TB/s, C4096
// T8192 48-51 us (5.3 TB/s, partly from the memory-side cache), 16 rows of 4096 5 us; backward C2048 T24960 with its column sums
// 128-141 us = 4.4-4.8 TB/s, of which the column kernel is 8.
#include <type_traits>

#include "contraction_kernel.hpp"
#include "train.hpp"

namespace tracea_amd {

namespace {

constexpr int V = 8;  // channels of a thread

template <typename T>
struct alignas(16) Eight {
  T x[V];
};

// Channel of a thread's element e: 8 in a row, or, where rows are not on 16 bytes, one apart between neighbouring lanes.
template <bool VEC>
__device__ __forceinline__ int channel(int e, int lane, int lanes) {
  return VEC ? lane * V + e : e * lanes + lane;
}
// A thread's channels of a row as they lie in memory: the next row's are requested before this one's are worked on.  One by one, every
// 16-bit value has a register of its own, and hold() keeps the conversions behind all loads: the compiler moves each of them behind
// its load's test of the channel, where it waits for that load (backward C2047 T24960 bf16 150 us, 452 without; C2048, in pieces of 16 bytes, 141 on that card).
template <typename T, bool VEC>
struct Loaded {
  Eight<T> p;
};
template <typename T>
struct Loaded<T, false> {
  std::conditional_t<sizeof(T) == 2, unsigned, float> x[V];
};
template <typename T, bool VEC>
__device__ __forceinline__ Loaded<T, VEC> request(const T *row, int lane, int lanes, int C) {
  Loaded<T, VEC> r;
  if constexpr (VEC) {
    const int c = channel<VEC>(0, lane, lanes);
    if (c < C) return {*(const Eight<T> *)(row + c)};
#pragma unroll
    for (int e = 0; e < V; ++e) r.p.x[e] = (T)0.0f;
  } else {
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const int c = channel<VEC>(e, lane, lanes);
      if constexpr (sizeof(T) == 2) r.x[e] = c < C ? ((const unsigned short *)row)[c] : 0u;
      else r.x[e] = c < C ? row[c] : 0.0f;
    }
  }
  return r;
}
template <typename T>
__device__ __forceinline__ void hold(Loaded<T, false> &r) {
#pragma unroll
  for (int e = 0; e < V; ++e) asm volatile("" : "+v"(r.x[e]));
}
template <typename T, bool VEC>
__device__ __forceinline__ void widen(const Loaded<T, VEC> &r, float (&x)[V]) {
#pragma unroll
  for (int e = 0; e < V; ++e) {
    if constexpr (VEC) {
      x[e] = (float)r.p.x[e];
    } else {
      if constexpr (sizeof(T) == 2) x[e] = (float)__builtin_bit_cast(T, (unsigned short)r.x[e]);
      else x[e] = r.x[e];
    }
  }
}
template <typename T, bool VEC>
__device__ __forceinline__ void store(T *row, int lane, int lanes, int C, const float (&x)[V]) {
  if constexpr (VEC) {
    const int c = channel<VEC>(0, lane, lanes);
    if (c < C) {
      Eight<T> p;
#pragma unroll
      for (int e = 0; e < V; ++e) p.x[e] = (T)x[e];
      *(Eight<T> *)(row + c) = p;
    }
  } else {
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const int c = channel<VEC>(e, lane, lanes);
      if (c < C) row[c] = (T)x[e];
    }
  }
}
// fp32 vectors of C channels, on 16 bytes where the rows are; absent: ones
template <bool VEC>
__device__ __forceinline__ void load_weights(const float *w, int lane, int lanes, int C, float (&x)[V]) {
  if (w == nullptr) {
#pragma unroll
    for (int e = 0; e < V; ++e) x[e] = 1.0f;
    return;
  }
  widen<float, VEC>(request<float, VEC>(w, lane, lanes, C), x);
}

// Sums of N values over the threads that share a row: `lanes` lanes of a wave (a power of two up to 64), then the waves of
// the workgroup.  `buf` alternates between two halves, so that one barrier a call is enough.
template <int N>
struct RowSum {
  float *buf;  // [2][16][N]
  int turn = 0;
  __device__ __forceinline__ void operator()(float (&x)[N], int lanes, int waves) {
    for (int m = 1; m < (lanes < 64 ? lanes : 64); m <<= 1) {
#pragma unroll
      for (int i = 0; i < N; ++i) x[i] += __shfl_xor(x[i], m, 64);
    }
    if (lanes <= 64) return;
    float *b = buf + turn * 16 * N;
    turn ^= 1;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    if (lane == 0) {
#pragma unroll
      for (int i = 0; i < N; ++i) b[wave * N + i] = x[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = b[i];
    for (int w = 1; w < waves; ++w) {
#pragma unroll
      for (int i = 0; i < N; ++i) x[i] += b[w * N + i];
    }
  }
};

// Which row a thread works on: `lanes` threads share one, a workgroup has blockDim / lanes at a time.
struct Place {
  int lane, lanes, slot, slots, b, first, end;
};
__device__ __forceinline__ Place place(const NormArgs &a, int lanes) {
  Place p;
  p.lanes = lanes;
  p.lane = threadIdx.x % lanes;
  p.slot = threadIdx.x / lanes;
  p.slots = blockDim.x / lanes;
  p.b = blockIdx.y;
  p.first = blockIdx.x * a.rows_per_chunk;
  p.end = min(p.first + a.rows_per_chunk, a.T);
  return p;
}
template <typename T>
__device__ __forceinline__ T *row_of(const RowView &v, int b, int t) {
  return (T *)v.p + (long long)b * v.sb + (long long)t * v.ss;
}

template <typename T, bool VEC, bool POST, bool PRE>
__global__ void __launch_bounds__(1024) norm_forward_kernel(const NormArgs a, int lanes) {
  __shared__ float buf[2 * 16 * 2];
  const Place p = place(a, lanes);
  const int waves = blockDim.x >> 6;
  RowSum<1> row_sum{buf};
  if (p.first >= p.end) return;
  Loaded<T, VEC> next_x, next_h;
  auto fetch = [&](int t) __attribute__((always_inline)) {
    const int tt = t < p.end ? t : p.first;
    next_x = request<T, VEC>(row_of<const T>(a.x, p.b, tt), p.lane, lanes, a.C);
    if constexpr (POST) next_h = request<T, VEC>(row_of<const T>(a.h, p.b, tt), p.lane, lanes, a.C);
  };
  fetch(p.first + p.slot);
  float gw[V], wp[V];  // gate * w_post, w_pre
  if constexpr (POST) {
    float gate[V];
    load_weights<VEC>(a.w_post, p.lane, lanes, a.C, gw);
    load_weights<VEC>(a.gate == nullptr ? nullptr : a.gate + p.b * a.gate_sb, p.lane, lanes, a.C, gate);
#pragma unroll
    for (int e = 0; e < V; ++e) gw[e] *= gate[e];
  }
  if constexpr (PRE) load_weights<VEC>(a.w_pre, p.lane, lanes, a.C, wp);
  const float per_c = 1.0f / (float)a.C;
  for (int t0 = p.first; t0 < p.end; t0 += p.slots) {  // (every thread takes every turn: there is a barrier in it)
    const int tt = t0 + p.slot;
    const bool there = tt < p.end;
    float x[V], h[V];
    widen<T, VEC>(next_x, x);
    if constexpr (POST) widen<T, VEC>(next_h, h);
    if (t0 + p.slots < p.end) fetch(tt + p.slots);
    if constexpr (POST) {
      float sum[1] = {0.0f};
#pragma unroll
      for (int e = 0; e < V; ++e) sum[0] = __builtin_fmaf(h[e], h[e], sum[0]);
      row_sum(sum, lanes, waves);
      const float r1 = rsqrtf(sum[0] * per_c + a.eps);
#pragma unroll
      for (int e = 0; e < V; ++e) x[e] = a.scale * x[e] + (h[e] * r1) * gw[e];
      if (there) store<T, VEC>(row_of<T>(a.x_out, p.b, tt), p.lane, lanes, a.C, x);
    }
    if constexpr (PRE) {
      float sum[1] = {0.0f};
#pragma unroll
      for (int e = 0; e < V; ++e) sum[0] = __builtin_fmaf(x[e], x[e], sum[0]);
      row_sum(sum, lanes, waves);
      const float r2 = rsqrtf(sum[0] * per_c + a.eps);
#pragma unroll
      for (int e = 0; e < V; ++e) x[e] = x[e] * r2 * wp[e];
      if (there) store<T, VEC>(row_of<T>(a.y, p.b, tt), p.lane, lanes, a.C, x);
    }
  }
}

template <typename T, bool VEC, bool POST, bool PRE>
__global__ void __launch_bounds__(1024) norm_backward_kernel(const NormArgs a, int lanes) {
  __shared__ float buf[2 * 16 * 6];
  const Place p = place(a, lanes);
  const int waves = blockDim.x >> 6;
  RowSum<6> row_sum{buf};
  const bool has_dx = a.dx_out.p != nullptr;
  constexpr bool AHEAD = VEC && sizeof(T) == 2;  // (else a row more takes the registers beyond the 128 that 1024 threads have)
  Loaded<T, VEC> next_x, next_g, next_h, next_d;
  auto fetch = [&](int t) __attribute__((always_inline)) {
    const int tt = t < p.end ? t : p.first;
    if constexpr (PRE) {
      next_x = request<T, VEC>(row_of<const T>(a.x_out, p.b, tt), p.lane, lanes, a.C);
      next_g = request<T, VEC>(row_of<const T>(a.dy, p.b, tt), p.lane, lanes, a.C);
    }
    if constexpr (POST) next_h = request<T, VEC>(row_of<const T>(a.h, p.b, tt), p.lane, lanes, a.C);
    if (has_dx) next_d = request<T, VEC>(row_of<const T>(a.dx_out, p.b, tt), p.lane, lanes, a.C);
  };
#pragma unroll
  for (int e = 0; e < V; ++e) {
    if constexpr (VEC) next_d.p.x[e] = (T)0.0f;
    else next_d.x[e] = 0;
  }
  if (AHEAD && p.first < p.end) fetch(p.first + p.slot);
  float gw[V], wp[V], sa[V], sp[V];
  if constexpr (POST) {
    float gate[V];
    load_weights<VEC>(a.w_post, p.lane, lanes, a.C, gw);
    load_weights<VEC>(a.gate == nullptr ? nullptr : a.gate + p.b * a.gate_sb, p.lane, lanes, a.C, gate);
#pragma unroll
    for (int e = 0; e < V; ++e) gw[e] *= gate[e];
  }
  if constexpr (PRE) load_weights<VEC>(a.w_pre, p.lane, lanes, a.C, wp);
#pragma unroll
  for (int e = 0; e < V; ++e) sa[e] = sp[e] = 0.0f;
  const float per_c = 1.0f / (float)a.C;
  for (int t0 = p.first; t0 < p.end; t0 += p.slots) {
    const int tt = t0 + p.slot;
    const bool there = tt < p.end;
    float x[V], g[V], h[V], d[V];
    if constexpr (!AHEAD) fetch(tt);
    if constexpr (!AHEAD && sizeof(T) == 2) {  // (32-bit values have no conversions)
      if constexpr (PRE) {
        hold(next_x);
        hold(next_g);
      }
      if constexpr (POST) hold(next_h);
      hold(next_d);
    }
    if constexpr (PRE) {
      widen<T, VEC>(next_x, x);
      widen<T, VEC>(next_g, g);
    }
    if constexpr (POST) widen<T, VEC>(next_h, h);
    widen<T, VEC>(next_d, d);
    if (AHEAD && t0 + p.slots < p.end) fetch(tt + p.slots);
    // x'.x', g.x', h.h, and (gate w_post h).dx', .g, .x': mean(a h^) follows from the last three
    float s[6] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int e = 0; e < V; ++e) {
      if constexpr (PRE) {
        const float gv = g[e] * wp[e];
        s[0] = __builtin_fmaf(x[e], x[e], s[0]);
        s[1] = __builtin_fmaf(gv, x[e], s[1]);
      }
      if constexpr (POST) {
        const float f = gw[e] * h[e];
        s[2] = __builtin_fmaf(h[e], h[e], s[2]);
        s[3] = __builtin_fmaf(f, d[e], s[3]);
        if constexpr (PRE) {
          s[4] = __builtin_fmaf(f, g[e] * wp[e], s[4]);
          s[5] = __builtin_fmaf(f, x[e], s[5]);
        }
      }
    }
    row_sum(s, lanes, waves);
    const float r2 = PRE ? rsqrtf(s[0] * per_c + a.eps) : 0.0f;
    const float m2 = PRE ? s[1] * r2 * per_c : 0.0f;  // mean(g x^)
    const float r1 = POST ? rsqrtf(s[2] * per_c + a.eps) : 0.0f;
    const float m1 = POST ? (s[3] + r2 * (s[4] - r2 * m2 * s[5])) * r1 * per_c : 0.0f;  // mean(a h^)
    float o[V];
#pragma unroll
    for (int e = 0; e < V; ++e) {
      float dt = d[e];
      if constexpr (PRE) {
        const float xn = x[e] * r2;
        dt += r2 * (g[e] * wp[e] - xn * m2);
        sp[e] = there ? __builtin_fmaf(g[e], xn, sp[e]) : sp[e];
      }
      o[e] = POST ? a.scale * dt : dt;
      if constexpr (POST) {
        const float hn = h[e] * r1;
        sa[e] = there ? __builtin_fmaf(dt, hn, sa[e]) : sa[e];
        h[e] = r1 * (dt * gw[e] - hn * m1);
      }
    }
    if (there) {
      store<T, VEC>(row_of<T>(a.dx, p.b, tt), p.lane, lanes, a.C, o);
      if constexpr (POST) {
        if (a.dh.p != nullptr) store<T, VEC>(row_of<T>(a.dh, p.b, tt), p.lane, lanes, a.C, h);
      }
    }
  }
  if (a.partial == nullptr) return;
  // rows side by side in a wave: their column sums first, in the order of the slots' halves
  for (int m = lanes; m < 64; m <<= 1) {
#pragma unroll
    for (int e = 0; e < V; ++e) {
      sa[e] += __shfl_xor(sa[e], m, 64);
      sp[e] += __shfl_xor(sp[e], m, 64);
    }
  }
  if (lanes < 64 && (threadIdx.x & 63) >= (unsigned)lanes) return;
  const long long plane = (long long)gridDim.y * gridDim.x * a.C;
  float *out = a.partial + ((long long)p.b * gridDim.x + blockIdx.x) * a.C;
#pragma unroll
  for (int e = 0; e < V; ++e) {
    const int c = channel<VEC>(e, p.lane, lanes);
    if (c < a.C) {
      if constexpr (POST) out[c] = sa[e];
      if constexpr (PRE) out[plane + c] = sp[e];
    }
  }
}

// Adds up the partial rows: a workgroup takes 16 channels of one sum (blockIdx.y: dw_post and the shared dgate, dw_pre, then dgate of each batch
// entry), 64 groups of threads a 64th of the rows each, in an order that does not change.
__global__ void __launch_bounds__(1024) norm_columns_kernel(const NormArgs a) {
  __shared__ float s_sum[64][16];
  const int cl = threadIdx.x & 15, group = threadIdx.x >> 4, c = blockIdx.x * 16 + cl, task = blockIdx.y;
  const int cc = min(c, a.C - 1);
  const bool shared_gate = a.gate_sb == 0;
  if (task == 0 ? a.dw_post == nullptr && (a.dgate == nullptr || !shared_gate) : task == 1 && a.dw_pre == nullptr) return;
  const float *rows = a.partial;
  long long n = (long long)a.B * a.chunks;
  if (task == 1) rows += n * a.C;
  if (task > 1) {
    rows += (long long)(task - 2) * a.chunks * a.C;
    n = a.chunks;
  }
  const bool weigh = task == 0 && a.gate != nullptr && !shared_gate;  // dw_post = sum over b of gate_b A_b
  float x = 0.0f;
  for (long long k = group; k < n; k += 64) {
    const float v = rows[k * a.C + cc];
    x = weigh ? __builtin_fmaf(a.gate[k / a.chunks * a.gate_sb + cc], v, x) : x + v;
  }
  s_sum[group][cl] = x;
  __syncthreads();
  if (group != 0 || c >= a.C) return;
  for (int g = 1; g < 64; ++g) x += s_sum[g][cl];
  if (task == 0) {
    if (a.dw_post != nullptr) a.dw_post[c] = a.gate != nullptr && shared_gate ? x * a.gate[c] : x;
    if (a.dgate != nullptr && shared_gate) a.dgate[c] = x * a.w_post[c];
  } else if (task == 1) {
    a.dw_pre[c] = x;
  } else {
    a.dgate[(long long)(task - 2) * a.gate_sb + c] = x * a.w_post[c];
  }
}

// Threads that share a row of C channels, 8 each: lanes of a wave up to 512 channels, else whole waves.
struct Shape {
  int lanes, threads;
};
Shape shape_of(int C) {
  const int pieces = (C + V - 1) / V;
  if (pieces > 32) {
    const int lanes = (pieces + 63) / 64 * 64;
    return {lanes, lanes};
  }
  int lanes = 1;
  while (lanes < pieces) lanes <<= 1;
  return {lanes, 64};
}

template <typename T, bool VEC>
int forward(const NormArgs &a, hipStream_t stream) {
  const Shape s = shape_of(a.C);
  const dim3 grid((unsigned)a.chunks, (unsigned)a.B), block((unsigned)s.threads);
  if (a.h.p != nullptr && a.y.p != nullptr) hipLaunchKernelGGL((norm_forward_kernel<T, VEC, true, true>), grid, block, 0, stream, a, s.lanes);
  else if (a.h.p != nullptr) hipLaunchKernelGGL((norm_forward_kernel<T, VEC, true, false>), grid, block, 0, stream, a, s.lanes);
  else hipLaunchKernelGGL((norm_forward_kernel<T, VEC, false, true>), grid, block, 0, stream, a, s.lanes);
  return (int)hipGetLastError();
}
template <typename T, bool VEC>
int backward(const NormArgs &a, hipStream_t stream) {
  const Shape s = shape_of(a.C);
  const dim3 grid((unsigned)a.chunks, (unsigned)a.B), block((unsigned)s.threads);
  if (a.h.p != nullptr && a.dy.p != nullptr) hipLaunchKernelGGL((norm_backward_kernel<T, VEC, true, true>), grid, block, 0, stream, a, s.lanes);
  else if (a.h.p != nullptr) hipLaunchKernelGGL((norm_backward_kernel<T, VEC, true, false>), grid, block, 0, stream, a, s.lanes);
  else hipLaunchKernelGGL((norm_backward_kernel<T, VEC, false, true>), grid, block, 0, stream, a, s.lanes);
  if (a.partial != nullptr) {
    const unsigned tasks = 2 + (a.dgate != nullptr && a.gate_sb != 0 ? (unsigned)a.B : 0);
    hipLaunchKernelGGL(norm_columns_kernel, dim3((unsigned)((a.C + 15) / 16), tasks), dim3(1024), 0, stream, a);
  }
  return (int)hipGetLastError();
}
template <typename T>
int any(const NormArgs &a, bool back, hipStream_t stream) {
  if (back) return a.vec ? backward<T, true>(a, stream) : backward<T, false>(a, stream);
  return a.vec ? forward<T, true>(a, stream) : forward<T, false>(a, stream);
}

}  // namespace

// Workgroups per batch entry: one round of them.  Of waves on a CU, forward 20 (GPU time of a call, us, one card: C4096 T8192 bf16 51, with 12
// 75; C1152 T8192 f16 22.1, with 16 23.7, with 32 19.5; C2048 T24960 91-93 with any), backward 12 where a row takes up to four waves,
// 16 beyond (C2048 T24960 bf16 141, with 16 145, with 8 137; C2047 150, with 8 171; C1152 43.5, with 8 54; C4096 T8192 101, with 12
// 99).  Backward a workgroup has at least four rows, or its partial column sums are a good part of what it moves (C1001 T999 f32 18.8;
// one row each 21.7).
int norm_chunks(int B, int T, int C, int cus, bool backward) {
  const Shape s = shape_of(C);
  const int slots = s.threads / s.lanes;  // rows a workgroup has at a time
  const int waves = s.threads / 64, on_cu = (backward ? (waves <= 4 ? 12 : 16) : 20) / waves;
  const long long want = (long long)cus * (on_cu > 1 ? on_cu : 1) / B;
  const long long least_rows = backward ? 4ll * slots : slots, most = (T + least_rows - 1) / least_rows;
  const long long chunks = want < most ? want : most;
  return chunks < 1 ? 1 : (int)chunks;
}

int launch_norm_forward(const NormArgs &a, int dtype, hipStream_t stream) {
  return dtype == DT_F32 ? any<float>(a, false, stream) : dtype == DT_F16 ? any<_Float16>(a, false, stream) : any<__bf16>(a, false, stream);
}
int launch_norm_backward(const NormArgs &a, int dtype, hipStream_t stream) {
  return dtype == DT_F32 ? any<float>(a, true, stream) : dtype == DT_F16 ? any<_Float16>(a, true, stream) : any<__bf16>(a, true, stream);
}

}  // namespace tracea_amd
