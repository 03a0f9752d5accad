// A caller's tensor views and the device they live on, as the dispatch files read them.
#pragma once
#include <algorithm>

#include "dispatch.hpp"

namespace tracea_amd {

struct View {
  void *ptr = nullptr;
  int rank = 0;
  long long shape[4] = {0, 0, 0, 0};
  long long stride[4] = {0, 0, 0, 0};
  int dtype = 0;
  int device = -1;
};

// Copies a TraceaTensorView; a NULL stride array means contiguous row-major.
inline TraceaStatus read_view(const char *what, const TraceaTensorView &t, int want_rank, View *v) {
  if (t.ptr == nullptr) return fail(TRACEA_INVALID_PARAMS, "%s: data pointer is NULL", what);
  if (t.shape == nullptr) return fail(TRACEA_INVALID_PARAMS, "%s: shape pointer is NULL", what);
  if ((int)t.rank != want_rank)
    return fail(TRACEA_INVALID_PARAMS, "%s: expected rank %d, got %u", what, want_rank, t.rank);
  v->ptr = t.ptr;
  v->rank = (int)t.rank;
  for (int i = 0; i < want_rank; ++i) v->shape[i] = (long long)t.shape[i];
  if (t.stride != nullptr) {
    for (int i = 0; i < want_rank; ++i) v->stride[i] = (long long)t.stride[i];
  } else {
    long long s = 1;
    for (int i = want_rank - 1; i >= 0; --i) {
      v->stride[i] = s;
      s *= v->shape[i];
    }
  }
  v->dtype = (int)t.dtype;
  v->device = t.device_id;
  return TRACEA_SUCCESS;
}

inline bool is_half(int dt) { return dt == TRACEA_DTYPE_FLOAT16 || dt == TRACEA_DTYPE_BFLOAT16; }
inline bool is_float_type(int dt) { return dt == TRACEA_DTYPE_FLOAT32 || is_half(dt); }
inline int elem_size(int dt) { return dt == TRACEA_DTYPE_FLOAT32 || dt == TRACEA_DTYPE_INT32 ? 4 : dt == TRACEA_DTYPE_INT8 ? 1 : 2; }
inline bool aligned(const void *p, size_t a) { return (((uintptr_t)p) & (a - 1)) == 0; }

// Rows of equal length on one pitch, the form of most views: element rows `pitch` apart, `len` elements of each used.
inline bool row_form(const View &v, long long *pitch, long long *len) {
  if (v.rank < 2 || v.stride[v.rank - 1] != 1) return false;
  // the pitch is the stride of the last dim but one; a [B,H,S,D] view of [B,S,H,D] storage has its heads inside the row
  *pitch = v.stride[v.rank - 2];
  *len = v.shape[v.rank - 1];
  if (*pitch < *len) return false;
  for (int i = v.rank - 3; i >= 0; --i) {
    if (v.shape[i] == 1 || v.stride[i] % *pitch == 0) continue;
    if (v.stride[i] < *len || (*len += (v.shape[i] - 1) * v.stride[i]) > *pitch) return false;
  }
  return true;
}

// Whether no sum of d_i * stride_i, first_i <= d_i <= last_i, strides from the `n`-th on descending, is `rest` (elements).  Gives up (false)
// where more than a few d_i come into question, which the strides of a tensor's own layout do not allow.
struct Steps {
  long long stride, first, last;
};
inline bool unreachable(const Steps *s, int n, long long rest) {
  if (n == 0) return rest != 0;
  long long low = 0, high = 0;  // what the smaller strides reach
  for (int i = 1; i < n; ++i) {
    low += s[i].first * s[i].stride;
    high += s[i].last * s[i].stride;
  }
  auto floor_div = [](long long x, long long y) { return x / y - (x % y < 0); };
  const long long from = std::max(s->first, -floor_div(high - rest, s->stride)), to = std::min(s->last, floor_div(rest - low, s->stride));
  if (to - from >= 4) return false;
  for (long long d = from; d <= to; ++d)
    if (!unreachable(s + 1, n - 1, rest - d * s->stride)) return false;
  return true;
}
// Two views with the same strides: slots of one buffer, whatever lies between their rows and heads.
inline bool slots_apart(const View &a, const View &b) {
  const long long size = elem_size(a.dtype), apart = (long long)((intptr_t)b.ptr - (intptr_t)a.ptr);
  if (a.rank != b.rank || size != elem_size(b.dtype) || apart % size != 0) return false;
  Steps s[4];
  int n = 0;
  for (int i = 0; i < a.rank; ++i) {
    if (a.shape[i] == 1 && b.shape[i] == 1) continue;
    const long long step = a.shape[i] > 1 ? a.stride[i] : b.stride[i];
    if (a.shape[i] > 1 && b.shape[i] > 1 && a.stride[i] != b.stride[i]) return false;
    if (step > 0) s[n++] = {step, 1 - b.shape[i], a.shape[i] - 1};
    else if (step < 0) s[n++] = {-step, 1 - a.shape[i], b.shape[i] - 1};
  }
  std::sort(s, s + n, [](const Steps &x, const Steps &y) { return x.stride > y.stride; });
  return unreachable(s, n, apart / size);
}

// Whether two views may share an element (columns of one buffer side by side, a query tensor inside a packed
// [Q K V] row or head and the like are told apart).
inline bool may_overlap(const View &a, const View &b) {
  auto span = [](const View &v, uintptr_t *lo, uintptr_t *hi) {
    long long first = 0, last = 0;
    for (int i = 0; i < v.rank; ++i) {
      if (v.shape[i] <= 0) return false;
      (v.stride[i] < 0 ? first : last) += (v.shape[i] - 1) * v.stride[i];
    }
    *lo = (uintptr_t)v.ptr + (uintptr_t)(first * elem_size(v.dtype));
    *hi = (uintptr_t)v.ptr + (uintptr_t)((last + 1) * elem_size(v.dtype));
    return true;
  };
  uintptr_t alo, ahi, blo, bhi;
  if (!span(a, &alo, &ahi) || !span(b, &blo, &bhi) || ahi <= blo || bhi <= alo) return false;
  long long pa, la, pb, lb;
  if (row_form(a, &pa, &la) && row_form(b, &pb, &lb)) {
    pa *= elem_size(a.dtype); la *= elem_size(a.dtype); pb *= elem_size(b.dtype); lb *= elem_size(b.dtype);
    long long d = ((long long)((intptr_t)b.ptr - (intptr_t)a.ptr)) % pa;
    if (d < 0) d += pa;
    if (pa == pb && d >= la && d + lb <= pa) return false;
  }
  return !slots_apart(a, b);
}

inline const char *dtype_name(int dt) {
  switch (dt) {
    case TRACEA_DTYPE_FLOAT32: return "f32";
    case TRACEA_DTYPE_FLOAT16: return "f16";
    case TRACEA_DTYPE_BFLOAT16: return "bf16";
    case TRACEA_DTYPE_INT32: return "i32";
    case TRACEA_DTYPE_INT8: return "i8";
    default: return "?";
  }
}

inline TraceaStatus check_device(const char *what, int device) {
  if (device < 0)
    return fail(TRACEA_CPU_ERROR,
                "%s: host memory (device_id -1) is not supported; this library has no CPU arm",
                what);
  if (device >= runtime_device_count())
    return fail(TRACEA_INVALID_PARAMS, "%s: device_id %d out of range (%d devices)", what, device,
                runtime_device_count());
  return TRACEA_SUCCESS;
}

// Makes `device` current for the lifetime of the object.
struct DeviceScope {
  int prev = -1;
  bool switched = false;
  hipError_t err = hipSuccess;
  explicit DeviceScope(int device) {
    err = hipGetDevice(&prev);
    if (err == hipSuccess && prev != device) {
      err = hipSetDevice(device);
      switched = err == hipSuccess;
    }
  }
  ~DeviceScope() {
    if (switched) (void)hipSetDevice(prev);
  }
};

inline TraceaStatus hip_status(const char *what, int e) {
  if (e == 0) return TRACEA_SUCCESS;
  return fail(TRACEA_CUDA_ERROR, "%s: %s", what, hipGetErrorString((hipError_t)e));
}

}  // namespace tracea_amd
