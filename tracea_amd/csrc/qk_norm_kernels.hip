// Norms of heads and rotary positions in one pass, gfx950, and its backward pass.
//   forward   y = R (x r w), r = rsqrt(mean of squares + eps) over a head's D values, R the rotation of rotary_kernels.hip
//   backward  dn = R^T dy, g = dn w, dx = r (g - x^ mean(g x^)), x^ = x r; dw = sum over all rows of dn x^
//
// Bound by memory: every element is read once and written once.  A row (a head of a token) is held by a group of lanes, each
// with the two pieces of 16 bytes (8 or 4 where the sizes ask for it) that hold the partners of a pair, so that the rotation needs no exchange and
// the norm one sum over the group.  The sine and cosine of a pair are worked out once for the heads that a lane group has of a token.
// Forward, 24960 tokens of 32 + 8 heads of 128 columns in bf16: 97 us, 5.3 TB/s (a copy: 5.06).
// The backward pass recomputes r, takes both sums of a row at once, keeps the weights' gradients of its rows in registers, joins
// them per workgroup, and a second kernel adds the workgroups' up in their order.  8192 tokens of 32 + 8 heads: 63 us, of which 53 read and write
// (4.8 TB/s), 4 to 5 are the second kernel's; 1539 tokens of 12 + 12 heads of 64 columns in fp32 17 us: latency, two launches.
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
struct __attribute__((packed, aligned(4))) Floats {  // of a weight, wherever it begins
  float x[E];
};

// What a lane holds of a row: N pairs (u, v) of columns.  In pieces: N = E elements of u and of v; else (E 0), one by one, up to 4 pairs that are
// turned and 4 couples of columns that are not.
template <typename T, int E, bool ADJ>
struct Lane {
  static constexpr bool VEC = E > 0;
  static constexpr int N = VEC ? E : 8;
  int at_u, at_v;  // pieces
  bool there, turned;
  int lane, D, P;

  __device__ __forceinline__ Lane(int lane_, int D_, int P_) : lane(lane_), D(D_), P(P_) {
    if constexpr (VEC) {
      const int pieces = P / E;
      there = lane * 2 * E < D;
      turned = lane < pieces;
      at_u = turned ? (ADJ ? 2 * lane * E : lane * E) : 2 * P + (lane - pieces) * 2 * E;
      at_v = turned && !ADJ ? at_u + P : at_u + E;
      if (!there) at_u = at_v = 0;
    }
  }
  // columns of couple k, and whether they are there (one by one)
  __device__ __forceinline__ void columns(int k, int &u, int &v, bool &has_u, bool &has_v) const {
    if (k < 4) {
      const int p = lane + 64 * k;
      u = ADJ ? 2 * p : p;
      v = ADJ ? 2 * p + 1 : p + P;
      has_u = has_v = p < P;
    } else {
      u = 2 * P + lane + 128 * (k - 4);
      v = u + 64;
      has_u = u < D;
      has_v = v < D;
    }
  }
  template <typename F>
  __device__ __forceinline__ void load(const F *row, float (&u)[N], float (&v)[N]) const {
    if constexpr (VEC) {
#pragma unroll
      for (int e = 0; e < N; ++e) u[e] = v[e] = 0.0f;
      if (there) {
        const Piece<F, E> a = *(const Piece<F, E> *)(row + at_u), b = *(const Piece<F, E> *)(row + at_v);
        couple(a.x, b.x, u, v);
      }
    } else {
#pragma unroll
      for (int k = 0; k < N; ++k) {
        int cu, cv;
        bool hu, hv;
        columns(k, cu, cv, hu, hv);
        u[k] = hu ? (float)row[cu] : 0.0f;
        v[k] = hv ? (float)row[cv] : 0.0f;
      }
    }
  }
  __device__ __forceinline__ void load_weight(const float *w, float (&u)[N], float (&v)[N]) const {
    if constexpr (VEC) {
#pragma unroll
      for (int e = 0; e < N; ++e) u[e] = v[e] = 0.0f;
      if (there) {
        const Floats<E> a = *(const Floats<E> *)(w + at_u), b = *(const Floats<E> *)(w + at_v);
        couple(a.x, b.x, u, v);
      }
    } else {
      load(w, u, v);
    }
  }
  // The partners of pairs side by side lie in one piece: the first half of the pairs in a, the second in b.
  template <typename A, typename B>
  __device__ __forceinline__ void couple(const A &a, const A &b, B &u, B &v) const {
#pragma unroll
    for (int e = 0; e < E; ++e) {
      if constexpr (ADJ) {
        u[e] = (float)(e < E / 2 ? a : b)[2 * (e % (E / 2))];
        v[e] = (float)(e < E / 2 ? a : b)[2 * (e % (E / 2)) + 1];
      } else {
        u[e] = (float)a[e];
        v[e] = (float)b[e];
      }
    }
  }
  // A row as it lies in memory: requested before the one ahead of it is worked on (in pieces; one by one, rows are not requested ahead).
  struct Raw {
    Piece<T, VEC ? E : 1> a, b;
  };
  __device__ __forceinline__ void request(const T *row, Raw &r) const {
    if constexpr (VEC) {
      if (there) {
        r.a = *(const Piece<T, E> *)(row + at_u);
        r.b = *(const Piece<T, E> *)(row + at_v);
      }
    }
  }
  __device__ __forceinline__ void take(const T *row, const Raw &r, float (&u)[N], float (&v)[N]) const {
    if constexpr (VEC) {
#pragma unroll
      for (int e = 0; e < N; ++e) u[e] = v[e] = 0.0f;
      if (there) couple(r.a.x, r.b.x, u, v);
    } else {
      load(row, u, v);
    }
  }
  template <typename F>
  __device__ __forceinline__ void store(F *row, const float (&u)[N], const float (&v)[N]) const {
    if constexpr (VEC) {
      if (!there) return;
      Piece<F, E> a, b;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        if constexpr (ADJ) {
          (e < E / 2 ? a : b).x[2 * (e % (E / 2))] = (F)u[e];
          (e < E / 2 ? a : b).x[2 * (e % (E / 2)) + 1] = (F)v[e];
        } else {
          a.x[e] = (F)u[e];
          b.x[e] = (F)v[e];
        }
      }
      *(Piece<F, E> *)(row + at_u) = a;
      *(Piece<F, E> *)(row + at_v) = b;
    } else {
#pragma unroll
      for (int k = 0; k < N; ++k) {
        int cu, cv;
        bool hu, hv;
        columns(k, cu, cv, hu, hv);
        if (hu) row[cu] = (F)u[k];
        if (hv) row[cv] = (F)v[k];
      }
    }
  }
  __device__ __forceinline__ bool is_turned(int k) const { return VEC ? turned : k < 4; }
  __device__ __forceinline__ int pair(int k) const { return VEC ? lane * E + k : lane + 64 * k; }

  __device__ __forceinline__ void angles(const QkNormArgs &a, int b, int s, float (&c)[N], float (&sn)[N]) const {
#pragma unroll
    for (int k = 0; k < N; ++k) {
      c[k] = 1.0f;
      sn[k] = 0.0f;
    }
    if (P == 0 || (VEC && !turned)) return;
    const int *pos = a.positions + b * a.pos_sb + s * a.pos_ss;
#pragma unroll
    for (int k = 0; k < (VEC ? N : 4); ++k) {
      const int p = pair(k);
      if (!VEC && p >= P) continue;
      int axis = 0;
      for (int x = 1; x < a.axes; ++x) axis += p >= a.first[x];
      turn(pos[axis], a.inv_freq[p], 1.0f, c[k], sn[k]);
    }
  }
};

__device__ __forceinline__ float group_sum(float x, int lanes) {
  for (int m = 1; m < lanes; m <<= 1) x += __shfl_xor(x, m, 64);
  return x;
}

template <typename T>
__device__ __forceinline__ T *row_of(const HeadView &t, int b, int h, int s) {
  return (T *)t.p + b * t.sb + h * t.sh + s * t.ss;
}

template <typename T, int E, bool ADJ>
__global__ void __launch_bounds__(256) qk_norm_forward_kernel(const QkNormArgs a) {
  using L = Lane<T, E, ADJ>;
  constexpr int N = L::N;
  const int groups = 256 / a.lanes, lane = threadIdx.x & (a.lanes - 1);
  const L me(lane, a.D, a.P);
  const long long item = ((long long)blockIdx.y * gridDim.x + blockIdx.x) * groups + threadIdx.x / a.lanes, token = item / a.beside;
  const int slot = (int)(item - token * a.beside);
  if (token >= (long long)a.B * a.S) return;
  const int b = (int)(token / a.S), s = (int)(token - (long long)b * a.S);
  float c[N], sn[N];
  me.angles(a, b, s, c, sn);
  int h = slot;
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    float wu[N], wv[N];
#pragma unroll
    for (int k = 0; k < N; ++k) wu[k] = wv[k] = 1.0f;
    if (a.w[t] != nullptr && h < a.H[t]) me.load_weight(a.w[t], wu, wv);
    for (; h < a.H[t]; h += a.beside) {
      float u[N], v[N];
      me.load(row_of<const T>(a.x[t], b, h, s), u, v);
      float ss = 0.0f;
#pragma unroll
      for (int k = 0; k < N; ++k) ss += u[k] * u[k] + v[k] * v[k];
      const float r = rsqrtf(group_sum(ss, a.lanes) * a.inv_d + a.eps);
#pragma unroll
      for (int k = 0; k < N; ++k) {
        const float nu = u[k] * r * wu[k], nv = v[k] * r * wv[k];
        u[k] = me.is_turned(k) ? nu * c[k] - nv * sn[k] : nu;
        v[k] = me.is_turned(k) ? nv * c[k] + nu * sn[k] : nv;
      }
      me.store(row_of<T>(a.out[t], b, h, s), u, v);
    }
    h -= a.H[t];
  }
}

template <typename T, int E, bool ADJ>
__global__ void __launch_bounds__(256) qk_norm_backward_kernel(const QkNormArgs a) {
  using L = Lane<T, E, ADJ>;
  constexpr int N = L::N;
  extern __shared__ float s_dw[];  // [lane groups][D]
  const int groups = 256 / a.lanes, lane = threadIdx.x & (a.lanes - 1), group = threadIdx.x / a.lanes;
  const L me(lane, a.D, a.P);
  const long long items = (long long)a.B * a.S * a.beside;
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    float wu[N], wv[N], du[N], dv[N];
#pragma unroll
    for (int k = 0; k < N; ++k) {
      wu[k] = wv[k] = 1.0f;
      du[k] = dv[k] = 0.0f;
    }
    if (a.w[t] != nullptr) me.load_weight(a.w[t], wu, wv);
    if (a.H[t] > 0)
      for (long long item = (long long)blockIdx.x * groups + group; item < items; item += (long long)gridDim.x * groups) {
        const long long token = item / a.beside;
        const int slot = (int)(item - token * a.beside), b = (int)(token / a.S), s = (int)(token - (long long)b * a.S);
        typename L::Raw x, dy, x_next, dy_next;
        if (slot < a.H[t]) {  // (on their way while the angles are worked out)
          me.request(row_of<const T>(a.x[t], b, slot, s), x);
          me.request(row_of<const T>(a.dout[t], b, slot, s), dy);
        }
        float c[N], sn[N];
        me.angles(a, b, s, c, sn);
        for (int h = slot; h < a.H[t]; h += a.beside, x = x_next, dy = dy_next) {
          if (h + a.beside < a.H[t]) {
            me.request(row_of<const T>(a.x[t], b, h + a.beside, s), x_next);
            me.request(row_of<const T>(a.dout[t], b, h + a.beside, s), dy_next);
          }
          float u[N], v[N], p[N], q[N];
          me.take(row_of<const T>(a.x[t], b, h, s), x, u, v);
          me.take(row_of<const T>(a.dout[t], b, h, s), dy, p, q);
          float ss = 0.0f, gx = 0.0f;
#pragma unroll
          for (int k = 0; k < N; ++k) {
            const float dnu = me.is_turned(k) ? p[k] * c[k] + q[k] * sn[k] : p[k], dnv = me.is_turned(k) ? q[k] * c[k] - p[k] * sn[k] : q[k];
            p[k] = dnu;
            q[k] = dnv;
            ss += u[k] * u[k] + v[k] * v[k];
            gx += dnu * wu[k] * u[k] + dnv * wv[k] * v[k];
          }
          for (int m = 1; m < a.lanes; m <<= 1) {
            ss += __shfl_xor(ss, m, 64);
            gx += __shfl_xor(gx, m, 64);
          }
          const float r = rsqrtf(ss * a.inv_d + a.eps), mean = gx * r * a.inv_d;  // of g x^
#pragma unroll
          for (int k = 0; k < N; ++k) {
            const float xu = u[k] * r, xv = v[k] * r;  // x^
            du[k] += p[k] * xu;
            dv[k] += q[k] * xv;
            u[k] = r * (p[k] * wu[k] - xu * mean);
            v[k] = r * (q[k] * wv[k] - xv * mean);
          }
          me.store(row_of<T>(a.out[t], b, h, s), u, v);
        }
      }
    if (a.dw[t] == nullptr) continue;
    __syncthreads();
    me.store(s_dw + group * a.D, du, dv);
    __syncthreads();
    for (int col = threadIdx.x; col < a.D; col += 256) {
      float sum = 0.0f;
      for (int g = 0; g < groups; ++g) sum += s_dw[g * a.D + col];
      a.partial[((long long)t * gridDim.x + blockIdx.x) * a.D + col] = sum;
    }
  }
}

// Sums over the workgroups: 16 columns of one weight, 64 runs of workgroups, whose loads are what it waits for (2048 workgroups, D128: 16 runs 8.3 us).
__global__ void __launch_bounds__(1024) qk_norm_weights_kernel(const QkNormArgs a) {
  constexpr int RUNS = 64;
  __shared__ float s_sum[RUNS][17];
  const int t = blockIdx.y, c16 = threadIdx.x & 15, run = threadIdx.x >> 4, col = blockIdx.x * 16 + c16;
  if (a.dw[t] == nullptr) return;
  float sum = 0.0f;
  if (col < a.D) {
#pragma unroll 8
    for (int i = run; i < a.blocks; i += RUNS) sum += a.partial[((long long)t * a.blocks + i) * a.D + col];
  }
  s_sum[run][c16] = sum;
  for (int half = RUNS / 2; half > 0; half >>= 1) {
    __syncthreads();
    if (run < half) s_sum[run][c16] += s_sum[run + half][c16];
  }
  if (run == 0 && col < a.D) a.dw[t][col] = s_sum[0][c16];
}

template <typename T, int E, bool ADJ>
int launch(const QkNormArgs &a, bool backward, hipStream_t stream) {
  const int groups = 256 / a.lanes;
  if (!backward) {
    // (at most 2^31 threads along x: a launch of 2^32 and more drops some of them without an error)
    const long long blocks = ((long long)a.B * a.S * a.beside + groups - 1) / groups, most = 1ll << 23, turns = (blocks + most - 1) / most;
    if (turns > 65535) return (int)hipErrorInvalidValue;
    hipLaunchKernelGGL((qk_norm_forward_kernel<T, E, ADJ>), dim3((unsigned)((blocks + turns - 1) / turns), (unsigned)turns), dim3(256), 0, stream, a);
    return (int)hipGetLastError();
  }
  hipLaunchKernelGGL((qk_norm_backward_kernel<T, E, ADJ>), dim3((unsigned)a.blocks), dim3(256), (unsigned)(groups * a.D * 4), stream, a);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || (a.dw[0] == nullptr && a.dw[1] == nullptr)) return (int)e;
  hipLaunchKernelGGL(qk_norm_weights_kernel, dim3((unsigned)((a.D + 15) / 16), 2), dim3(1024), 0, stream, a);
  return (int)hipGetLastError();
}
template <typename T>
int launch_type(const QkNormArgs &a, bool backward, hipStream_t stream) {
#define PIECES(E) \
  if (a.vec == E) return a.adjacent ? launch<T, E, true>(a, backward, stream) : launch<T, E, false>(a, backward, stream);
  if constexpr (sizeof(T) == 2) {
    PIECES(8)
  }
  PIECES(4)
  PIECES(2)
#undef PIECES
  return a.adjacent ? launch<T, 0, true>(a, backward, stream) : launch<T, 0, false>(a, backward, stream);
}
int launch_any(const QkNormArgs &a, int dtype, bool backward, hipStream_t stream) {
  if (dtype == DT_F32) return launch_type<float>(a, backward, stream);
  return dtype == DT_F16 ? launch_type<_Float16>(a, backward, stream) : launch_type<__bf16>(a, backward, stream);
}

}  // namespace

int launch_qk_norm_forward(const QkNormArgs &a, int dtype, hipStream_t stream) { return launch_any(a, dtype, false, stream); }
int launch_qk_norm_backward(const QkNormArgs &a, int dtype, hipStream_t stream) { return launch_any(a, dtype, true, stream); }

}  // namespace tracea_amd
