// Whether two views may share an element (csrc/host/views.hpp), against the elements themselves: random small views, counted out.
#include <cstdio>
#include <cstdlib>
#include <set>

#include "views.hpp"

using namespace tracea_amd;

static unsigned long long g_state = 12345;
static int below(int n) {
  g_state = g_state * 6364136223846793005ull + 1442695040888963407ull;
  return (int)((g_state >> 33) % (unsigned long long)n);
}

static char g_memory[1 << 16];
static int size_of(int dtype) { return dtype == TRACEA_DTYPE_FLOAT32 || dtype == TRACEA_DTYPE_INT32 ? 4 : 2; }

static View random_view(int dtype) {
  View v;
  v.rank = 1 + below(4);
  v.dtype = dtype;
  const int s = size_of(dtype);
  v.ptr = g_memory + (1 << 15) + (below(400) - 200) * s + (below(8) == 0 ? 1 + below(s) : 0);
  long long dense = 1;
  for (int i = v.rank - 1; i >= 0; --i) {
    v.shape[i] = 1 + below(4);
    v.stride[i] = below(3) ? dense * (1 + below(2)) + (below(3) == 0 ? below(3) : 0) : below(24) - 4;
    dense = dense * v.shape[i] + below(2) * below(5);
  }
  return v;
}

// As a slot of rows that hold several tensors: the form of packed operands and gradients, with heads inside or outside the slots.
static void packed_views(View *a, View *b, int dtype) {
  const int slots = 2 + below(3), d = 1 + below(5), h = 1 + below(3), s = 1 + below(4), n = 1 + below(3);
  const bool within_head = below(2) != 0;
  for (View *v : {a, b}) {
    v->rank = 4;
    v->dtype = dtype;
    const int slot = below(slots);
    v->ptr = g_memory + (1 << 15) + (slot * d * (within_head ? 1 : h) + (below(6) == 0 ? below(3) : 0)) * size_of(dtype);
    const long long head = (long long)d * (within_head ? slots : 1), row = (long long)slots * d * h;
    const long long shape[4] = {n, 1 + below(h), s, d}, stride[4] = {row * s, head, row, 1};
    for (int i = 0; i < 4; ++i) {
      v->shape[i] = shape[i];
      v->stride[i] = stride[i];
    }
  }
}

static std::set<long long> bytes_of(const View &v) {
  std::set<long long> all;
  const int e = size_of(v.dtype);
  long long n = 1;
  for (int i = 0; i < v.rank; ++i) n *= v.shape[i];
  for (long long k = 0; k < n; ++k) {
    long long rest = k, at = 0;
    for (int i = v.rank - 1; i >= 0; --i) {
      at += rest % v.shape[i] * v.stride[i];
      rest /= v.shape[i];
    }
    for (int j = 0; j < e; ++j) all.insert((char *)v.ptr - g_memory + at * e + j);
  }
  return all;
}
static bool share(const View &a, const View &b) {
  const std::set<long long> x = bytes_of(a), y = bytes_of(b);
  for (long long at : x)
    if (y.count(at)) return true;
  return false;
}

int main() {
  const int types[4] = {TRACEA_DTYPE_FLOAT32, TRACEA_DTYPE_FLOAT16, TRACEA_DTYPE_BFLOAT16, TRACEA_DTYPE_INT32};
  long missed = 0, apart = 0, told = 0, packed_apart = 0, packed_told = 0;
  for (int k = 0; k < 200000; ++k) {
    const bool packed = k % 2 != 0;
    View a, b;
    if (packed) {
      packed_views(&a, &b, types[below(4)]);
    } else {
      a = random_view(types[below(4)]);
      b = random_view(types[below(4)]);
    }
    const bool really = share(a, b), may = may_overlap(a, b);
    if (really && !may) ++missed;
    if (!really) {
      ++(packed ? packed_apart : apart);
      if (!may) ++(packed ? packed_told : told);
    }
  }
  printf("missed %ld, apart %ld of which told %ld, packed apart %ld of which told %ld\n", missed, apart, told, packed_apart, packed_told);
  return missed != 0;
}
