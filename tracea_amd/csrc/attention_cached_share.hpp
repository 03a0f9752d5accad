// What the kernels of attention over a cache share: how steps over keys are shared out between workgroups, and where pages lie.
//
// A problem is a block of rows of a (sequence, key/value head); its steps are runs of a.step keys.  What the workgroups have of them is worked
// out from the lengths on the device, in 32 bits (the host sees to that), whatever the lengths are.  Either every problem is cut into parts of
// the same number of steps by itself, a workgroup for each, where such parts are short (a.apart) and not more than the workgroups; or the
// steps of all problems, in the order (sequence, head, block), are one line, of which every workgroup has the same number.  A problem cut
// between workgroups leaves parts in the workspace: slot 2 w for a part that workgroup w begins with, 2 w + 1 for one that it comes to later;
// meta[problem] says which they are.
#pragma once
#include "attention_tile.hpp"
#include "cache.hpp"

namespace tracea_amd {

namespace {

__device__ __forceinline__ int query_of(const AttentionCachedArgs &a, int r) {
  return a.G == 1 ? r : (int)__umulhi((unsigned)r, a.g_magic);
}
__device__ __forceinline__ int keys_of(const AttentionCachedArgs &a, int b) {
  return min(max(a.k_len[b], 0), a.table.M * a.table.P);
}
__device__ __forceinline__ int queries_of(const AttentionCachedArgs &a, int b) {
  return a.q_len != nullptr ? min(max(a.q_len[b], 0), a.Sq) : a.Sq;
}
// Steps of a block of rows of sequence b: at least one, which writes what rows without keys get.
__device__ __forceinline__ int steps_of(const AttentionCachedArgs &a, int b) {
  return max(1, (keys_of(a, b) + a.step - 1) >> a.step_log2);
}

// A workgroup's share: `left` steps from step s0 of `inner` (head and block of rows) of sequence b, whose problems have sb steps.
struct Share {
  int b, inner, s0, sb, left;
  int first, per;  // where it begins in the line, or -1: a part of a problem cut by itself; steps of a share
};
__device__ __forceinline__ bool share_of(const AttentionCachedArgs &a, int lane, Share &w) {
  const int per_b = a.Hk * a.row_blocks, here = lane < a.B ? steps_of(a, lane) : 0;
  int steps, own, total, before = 0, mine;  // of lane l's sequence: steps and units of a problem, units in front of it
  auto scan = [&](int b0, int unit) __attribute__((always_inline)) {
    steps = b0 == 0 ? here : b0 + lane < a.B ? steps_of(a, b0 + lane) : 0;
    own = unit == 1 ? steps : (int)((unsigned)(steps + unit - 1) / (unsigned)unit);
    int x = own * per_b;
    mine = -x;
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) {
      const int y = __shfl_up(x, m, 64);
      x += lane >= m ? y : 0;
    }
    total = __builtin_amdgcn_readlane(x, 63);
    mine += x;
  };
  auto count = [&](int unit) __attribute__((always_inline)) {  // of all sequences; own, mine and total are left as the first 64 have them
    int n = 0;
    for (int b0 = (a.B - 1) & -64; b0 >= 0; b0 -= 64) {
      scan(b0, unit);
      n += total;
    }
    return n;
  };
  const int all = count(1);
  auto per_of = [&](int shares) { return (int)(((unsigned)all + (unsigned)shares - 1) / (unsigned)shares); };
  w.per = per_of(a.shares);
  if (w.per > a.twice) w.per = per_of(2 * a.shares);
  bool apart = w.per <= a.apart;
  if (apart) {
    const int parts = count(w.per);
    if ((int)blockIdx.x >= parts && parts <= a.workgroups) return false;
    apart = parts <= a.workgroups;
    if (!apart) (void)count(1);
  }
  if (!apart) w.per = per_of(a.line);
  if (!apart && (long long)blockIdx.x * w.per >= all) return false;
  const int at_unit = apart ? (int)blockIdx.x : (int)blockIdx.x * w.per, unit = apart ? w.per : 1;
  int b0 = 0;
  while (before + total <= at_unit) {
    before += total;
    b0 += 64;
    if (b0 >= a.B) return false;  // (lengths that somebody writes while they are read: the walk has to end)
    scan(b0, unit);
  }
  const int at = 63 - __clzll(__ballot(before + mine <= at_unit && own > 0));
  w.b = b0 + at;
  w.sb = __builtin_amdgcn_readlane(steps, at);
  const int u = at_unit - (before + __builtin_amdgcn_readlane(mine, at)), units = __builtin_amdgcn_readlane(own, at);
  w.inner = __builtin_amdgcn_readfirstlane((int)((unsigned)u / (unsigned)units));
  w.s0 = (u - w.inner * units) * unit;
  w.first = apart ? -1 : at_unit;
  w.left = apart ? min(w.per, w.sb - w.s0) : min(w.per, all - at_unit);
  return true;
}
// The next problem of the line.
__device__ __forceinline__ void next_problem(const AttentionCachedArgs &a, Share &w) {
  w.s0 = 0;
  if (++w.inner == a.Hk * a.row_blocks) {
    w.inner = 0;
    w.b = min(w.b + 1, a.B - 1);  // (the last only where lengths were changed meanwhile)
    w.sb = steps_of(a, w.b);
  }
}
// Who joins: the workgroup with a problem's first step writes its first slot and how many parts it has, or that it is not cut.
__device__ __forceinline__ void write_meta(const AttentionCachedArgs &a, const Share &w, int at, int n, bool begins) {
  const long long problem = (long long)w.b * a.Hk * a.row_blocks + w.inner;
  a.meta[2 * problem] = n == w.sb ? -1 : 2 * (int)blockIdx.x + (begins ? 0 : 1);
  a.meta[2 * problem + 1] = w.first < 0 ? (w.sb + w.per - 1) / w.per : (at + w.sb - 1) / w.per - (int)blockIdx.x + 1;
}

__device__ __forceinline__ float wave_max(float x) {
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) x = fmaxf(x, __shfl_xor(x, m, 64));
  return x;
}

// Where groups of 16 keys lie, one per lane: the first key's row of both caches in the head.
struct Places {
  unsigned k_lo, k_hi, v_lo, v_hi;
  unsigned long long valid;  // groups that have a page and a key

  // The places of the groups from `key` on (the lane's own); the lane's page, or 0, and whether it has one.
  __device__ __forceinline__ int locate(const AttentionCachedArgs &a, int b, int hk, int key, int end, bool &there) {
    const int group = key >> 4, slot = a.page_magic == 0 ? group : (int)__umulhi((unsigned)group, a.page_magic);
    int page = page_of(a.table, b, slot);  // (before the sequence's length has arrived)
    there = page >= 0 && key < end;
    const int place = there ? key - slot * a.table.P : 0;
    page = there ? page : 0;  // (something to load)
    const unsigned long long k = (unsigned long long)(a.k.p + page * a.k.sn + hk * a.k.sh + place * a.k.ss);
    const unsigned long long v = (unsigned long long)(a.v.p + page * a.v.sn + hk * a.v.sh + place * a.v.ss);
    k_lo = (unsigned)k; k_hi = (unsigned)(k >> 32);
    v_lo = (unsigned)v; v_hi = (unsigned)(v >> 32);
    valid = __ballot(there);
    return page;
  }
  static __device__ __forceinline__ const unsigned char *at(unsigned lo, unsigned hi, int e) {
    return (const unsigned char *)((unsigned long long)(unsigned)__builtin_amdgcn_readlane((int)lo, e) |
                                   (unsigned long long)(unsigned)__builtin_amdgcn_readlane((int)hi, e) << 32);
  }
  __device__ __forceinline__ const unsigned char *k(int e) const { return at(k_lo, k_hi, e); }
  __device__ __forceinline__ const unsigned char *v(int e) const { return at(v_lo, v_hi, e); }
};
__device__ __forceinline__ float of_lane(float x, int e) {
  return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, x), e));
}

// Two e4m3 codes of a register (its upper half: HI) times a power of two, in 16 bits: exact within the type's range, as e4m3 has no value that
// f16 or bf16 lacks.
template <int DT, bool HI>
__device__ __forceinline__ unsigned widen2(unsigned codes, float power = 1.0f) {
  if constexpr (DT == DT_F16) return __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)codes, power, HI));
  else return __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)codes, power, HI));
}
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

// 8 columns of a query from column c on, wherever the row begins.
__device__ __forceinline__ u32x4 query_columns(const AttentionCachedArgs &a, const unsigned short *row, bool there, int c) {
  u32x4 x = {0, 0, 0, 0};
  if (there && c < a.D) {
    if (a.q_vec) {
      x = *(const u32x4 *)(row + c);
    } else {
#pragma unroll
      for (int w = 0; w < 4; ++w) x[w] = (unsigned)row[c + 2 * w] | (unsigned)row[c + 2 * w + 1] << 16;
    }
  }
  return a.negate ? x ^ 0x80008000u : x;
}

}  // namespace

}  // namespace tracea_amd
