// What the dispatch files of the operators for training and of those over a key/value cache check of a call's operands, and the lock
// under which both launch what passes something on in a workspace.
#pragma once
#include <cstdlib>
#include <mutex>

#include "../train.hpp"
#include "views.hpp"

namespace tracea_amd {

// The launches of a call that pass something on in a workspace or in copies stay together on their stream, whichever threads use
// it: no other operator writes either buffer.
extern std::mutex g_launches;

inline TraceaStatus ready(const char *what) {
  return runtime_ready() ? TRACEA_SUCCESS : fail(TRACEA_UNKNOWN_ERROR, "%s: tracea_init has not been called", what);
}

inline long long count_of(const View &v) {
  long long n = 1;
  for (int i = 0; i < v.rank; ++i) n *= v.shape[i];
  return n;
}

// As read_view; a tensor without elements may have no address.
inline TraceaStatus read(const char *op, const char *name, const TraceaTensorView &t, int rank, View *v) {
  if (t.ptr != nullptr && t.shape != nullptr && (int)t.rank == rank) {  // (what can be read at all: no message has to be made up)
    const TraceaStatus st = read_view(name, t, rank, v);
    if (st != TRACEA_SUCCESS) return st;
  } else {
    char what[96];
    snprintf(what, sizeof(what), "%s: %s", op, name);
    TraceaTensorView u = t;
    static char nothing;
    if (u.ptr == nullptr && u.shape != nullptr && (int)u.rank == rank)
      for (int i = 0; i < rank; ++i)
        if (u.shape[i] == 0) u.ptr = &nothing;
    const TraceaStatus st = read_view(what, u, rank, v);
    if (st != TRACEA_SUCCESS) return st;
  }
  for (int i = 0; i < rank; ++i)
    if (t.shape[i] >= (1ull << 31)) return fail(TRACEA_UNSUPPORTED_CONFIG, "%s: %s: extents of 2^31 and more are not supported", op, name);
  return TRACEA_SUCCESS;
}

inline bool same_shape(const View &a, const View &b) {
  if (a.rank != b.rank) return false;
  for (int i = 0; i < a.rank; ++i)
    if (a.shape[i] != b.shape[i]) return false;
  return true;
}
inline bool same_view(const View &a, const View &b) {
  if (a.ptr != b.ptr || a.dtype != b.dtype || !same_shape(a, b)) return false;
  for (int i = 0; i < a.rank; ++i)
    if (a.shape[i] > 1 && a.stride[i] != b.stride[i]) return false;
  return true;
}
// A result whose elements may share an address (an expanded tensor and the like).
inline bool folds(const View &v) {
  long long reach = 0;  // of the dimensions with smaller strides
  bool used[4] = {false, false, false, false};
  for (int n = 0; n < v.rank; ++n) {
    int best = -1;
    for (int i = 0; i < v.rank; ++i)
      if (!used[i] && (best < 0 || std::llabs(v.stride[i]) < std::llabs(v.stride[best]))) best = i;
    used[best] = true;
    if (v.shape[best] <= 1) continue;
    if (std::llabs(v.stride[best]) <= reach) return true;
    reach += (v.shape[best] - 1) * std::llabs(v.stride[best]);
  }
  return false;
}

inline HeadView head_view(const View &v) { return HeadView{v.ptr, v.stride[0], v.stride[1], v.stride[2]}; }

inline TraceaStatus overlapping(const char *op, const char *what) {
  return fail(TRACEA_INVALID_PARAMS, "%s: %s", op, what);
}

}  // namespace tracea_amd
