// What the attention kernels that stream tiles of 64 rows through LDS share: the tiles' layout there, requests into it, reads of matrix
// operands from it, and the small parts of an online softmax.
#pragma once
#include "contraction_kernel.hpp"

namespace tracea_amd {

namespace {

constexpr int TILE = 64;  // rows of a streamed tile
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;
template <int DT>
__device__ __forceinline__ u32x4 pack_operand(const f32x4 &lo, const f32x4 &hi) {
  if constexpr (DT == DT_F16) {
    f16x8 h = {(_Float16)lo[0], (_Float16)lo[1], (_Float16)lo[2], (_Float16)lo[3],
               (_Float16)hi[0], (_Float16)hi[1], (_Float16)hi[2], (_Float16)hi[3]};
    return __builtin_bit_cast(u32x4, h);
  } else {
    bf16x8 h = {(__bf16)lo[0], (__bf16)lo[1], (__bf16)lo[2], (__bf16)lo[3],
                (__bf16)hi[0], (__bf16)hi[1], (__bf16)hi[2], (__bf16)hi[3]};
    return __builtin_bit_cast(u32x4, h);
  }
}
template <int DT>
__device__ __forceinline__ u32x2 pack_result(const f32x4 &x, float f) {
  if constexpr (DT == DT_F16) {
    f16x4 h = {(_Float16)(x[0] * f), (_Float16)(x[1] * f), (_Float16)(x[2] * f), (_Float16)(x[3] * f)};
    return __builtin_bit_cast(u32x2, h);
  } else {
    bf16x4 h = {(__bf16)(x[0] * f), (__bf16)(x[1] * f), (__bf16)(x[2] * f), (__bf16)(x[3] * f)};
    return __builtin_bit_cast(u32x2, h);
  }
}
// A tile in LDS: 64 rows of DL elements, the 16-byte column XOR-ed with a number f made of the row; 64 banks of 4 bytes, 16 lanes of
// 16 bytes or 32 of 8 at a time.  f serves both ways a tile is read:
//   row fragments (16 rows, four columns one apart): the hardware takes rows 0-3 and 12-15 of one column together with
//   rows 4-11 of the next, so that f of the former must be whole pairs {2n, 2n + 1};
//   transposing reads (8 rows x 2 columns): f / 2 must differ between rows 0-7, and between rows 8-15.
// (A plain rotation of the row has the second only: 128 of 368 LDS cycles of a pair of half-tiles were conflicts.)  With DL = 64
// two rows share a line of 256 bytes, and k is the line.
template <int DL>
struct Tile {
  static constexpr int ROW_BYTES = DL * 2, CH = DL / 8, RP = 256 / ROW_BYTES, BYTES = TILE * ROW_BYTES;
  static __device__ __forceinline__ int swz(int row) {
    const int k = (row / RP) & (CH - 1), upper = k / (CH / 2);
    return (((k & (CH / 2 - 1)) ^ (upper * (CH / 4))) << 1) | upper;
  }
};

// A direct-to-LDS load: lane l's bytes from its offset land at lds + l * size.  Written as instructions: behind the builtin
// the compiler, which cannot tell the buffers of a ring apart, waits for all requests in front of the next LDS read.  The
// kernels wait for a tile themselves (vmcnt(0) and a barrier) before they read it.  (s_nop: m0 is read by the load behind it; m0 is
// reserved, the compiler writes it in front of each use of its own.)
__device__ __forceinline__ void dma16(u32x4 rsrc, unsigned offset, unsigned lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(lds), "v"(offset), "s"(rsrc) : "memory");
}
__device__ __forceinline__ u32x4 resource(const void *base, unsigned bytes) {
  const unsigned long long at = (unsigned long long)base;
  return u32x4{(unsigned)__builtin_amdgcn_readfirstlane((int)(unsigned)at),
               (unsigned)__builtin_amdgcn_readfirstlane((int)(unsigned)(at >> 32)) & 0xffffu, bytes, 0x00020000u};
}
__device__ __forceinline__ unsigned lds_offset(const void *p) {
  return (unsigned)(unsigned long long)(__attribute__((address_space(3))) const void *)p;
}
__device__ __forceinline__ unsigned lds_address(const void *p) { return (unsigned)__builtin_amdgcn_readfirstlane((int)lds_offset(p)); }

// Requests 64 rows of a tensor into LDS, 16 bytes per lane and 1 KB per wave and request; a wave's requests are 16 (DL = 128) or 32 rows
// apart.  Columns from D on read as zeros.
constexpr unsigned BEYOND = 0x80000000u;  // an offset that no tile has: out of the resource's range, reads as zeros
// ... where the offset of row r + 16 is that of row r and a step, for whole tiles: offset(row) the byte offset of row 0..15 / 0..31 from `base`.
template <int DL, int WAVES, typename F>
__device__ __forceinline__ void load_tile(const void *base, long long step, const unsigned char *dst, int D, int lane, int wave_u, F &&offset) {
  using T = Tile<DL>;
  constexpr int RPI = 64 / T::CH, NI = TILE / (RPI * WAVES);
  const int first = wave_u * RPI, row = first + lane / T::CH;
  const int col = ((lane % T::CH) ^ T::swz(row)) << 3;
  const unsigned at = col >= D ? BEYOND : offset(row) + (unsigned)(col * 2), lds = lds_address(dst) + (unsigned)(first * T::ROW_BYTES);
#pragma unroll
  for (int i = 0; i < NI; ++i) dma16(resource((const char *)base + i * step, BEYOND), at, lds + (unsigned)(i * WAVES * RPI * T::ROW_BYTES));
}
// ... any rows: offset(row) is below 2^31, or BEYOND for a row that reads as zeros.
template <int DL, int WAVES, typename F>
__device__ __forceinline__ void load_tile_any(const void *base, const unsigned char *dst, int D, int lane, int wave_u, F &&offset) {
  using T = Tile<DL>;
  constexpr int RPI = 64 / T::CH, NI = TILE / (RPI * WAVES);
  const u32x4 rsrc = resource(base, BEYOND);
  const unsigned lds = lds_address(dst);
#pragma unroll
  for (int i = 0; i < NI; ++i) {
    const int first = (i * WAVES + wave_u) * RPI, row = first + lane / T::CH;
    const int col = ((lane % T::CH) ^ T::swz(row)) << 3;
    const unsigned off = offset(row);
    dma16(rsrc, (off == BEYOND || col >= D) ? BEYOND : off + (unsigned)(col * 2), lds + (unsigned)(first * T::ROW_BYTES));
  }
}

// Where a lane reads a tile, as LDS addresses: everything but the constant part of a fragment's place, which is XOR-ed in (it
// shares no bit with the row, and the bits that it shares with the swizzle are what the swizzle is for).
template <int DL>
__device__ __forceinline__ unsigned rows_base(const unsigned char *tile, int r16, int g4) {
  using T = Tile<DL>;
  return lds_offset(tile) + (unsigned)(r16 * T::ROW_BYTES + ((g4 ^ T::swz(r16)) << 4));
}
template <int DL>
__device__ __forceinline__ unsigned columns_base(const unsigned char *tile, int r16, int g4) {
  using T = Tile<DL>;
  const int row = g4 * 4 + (r16 >> 2);
  return lds_offset(tile) + (unsigned)(row * T::ROW_BYTES + ((((r16 & 3) >> 1) ^ T::swz(row)) << 4) + (r16 & 1) * 8);
}
typedef __attribute__((address_space(3))) const u32x4 lds_u32x4;
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
// First operand of a product over the head dimension: rows 16 rb .. + 15 of the tile, columns 32 ks .. + 31.
template <int DL>
__device__ __forceinline__ u32x4 read_rows(unsigned base, unsigned side, int rb, int ks) {
  return *(lds_u32x4 *)(uintptr_t)((base ^ (unsigned)(ks << 6)) + side + (unsigned)(rb * 16 * Tile<DL>::ROW_BYTES));
}
// First operand of a product over the rows 32 s .. + 31: columns 16 db .. + 15 of the tile, transposed.
template <int DL>
__device__ __forceinline__ u32x4 read_columns(unsigned base, unsigned side, int s, int db) {
  const unsigned at = (base ^ (unsigned)(db << 5)) + side + (unsigned)(s * 32 * Tile<DL>::ROW_BYTES);
  const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)(uintptr_t)at);
  const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)(uintptr_t)(at + 16 * Tile<DL>::ROW_BYTES));
  const u32x2 a = __builtin_bit_cast(u32x2, lo), b = __builtin_bit_cast(u32x2, hi);
  return u32x4{a[0], a[1], b[0], b[1]};
}

// Nothing is scheduled across: the compiler otherwise hoists the reads of several phases and runs out of registers.
__device__ __forceinline__ void fence() { __builtin_amdgcn_sched_barrier(0); }

// A value that the compiler takes for a new one: what follows from it is worked out again where it is used, in an instruction
// or two, instead of being held in registers all through a loop that has none to spare.
__device__ __forceinline__ unsigned fresh(unsigned x) {
  asm volatile("" : "+v"(x));
  return x;
}

// max / sum over the four 16-lane groups, through LDS
__device__ __forceinline__ float groups_max(float x) {
  x = fmaxf(x, __shfl_xor(x, 16, 64));
  return fmaxf(x, __shfl_xor(x, 32, 64));
}
__device__ __forceinline__ float groups_sum(float x) {
  x += __shfl_xor(x, 16, 64);
  return x + __shfl_xor(x, 32, 64);
}

// Consecutive workgroups go to the 8 XCDs in turn; handing each XCD a run of blocks brings a head's tiles into one L2.
__device__ __forceinline__ int xcd_run(int id, int total) {
  const int q = total >> 3, rem = total & 7, x = id & 7, i = id >> 3;
  return x * q + (x < rem ? x : rem) + i;
}

// A row's reference lies P_SHIFT powers of two below a score it has met and moves only when a tile exceeds that score by more than
// LAZY_MAX: a row needs one reference for all its keys, not the largest score.  Operands are up to 2^(P_SHIFT + LAZY_MAX), in f16
// 2^15; there the shift keeps what lies 2^25 below the largest probability (2^-25 is 0 in f16, 2^-14 its smallest normal number), of
// which a long row may have a tail that counts, and each key loses at most 2^-36 of the largest: nothing up to 2^24 keys.
template <int DT>
constexpr float P_SHIFT = DT == DT_F16 ? 11.0f : 0.0f;
template <int DT>
constexpr float LAZY_MAX = DT == DT_F16 ? 4.0f : 8.0f;

// Over a lane's own value and those of the other three 16-lane groups, by exchanges in the vector ALU: v_permlane16_swap trades the
// odd 16-lane rows of its first operand for the even ones of its second, v_permlane32_swap the halves; given one value
// twice, the two results are a lane's own and its partner's, in one order or the other.  (As instructions: the builtin hands back its first
// result twice.  The s_nop covers the wait between a vector-ALU write and the swap.)
__device__ __forceinline__ float groups_max_valu(float x) {
  float a0 = x, a1 = x;
  asm volatile("s_nop 1\n\tv_permlane16_swap_b32 %0, %1" : "+v"(a0), "+v"(a1));
  float b0 = fmaxf(a0, a1), b1 = b0;
  asm volatile("s_nop 1\n\tv_permlane32_swap_b32 %0, %1" : "+v"(b0), "+v"(b1));
  return fmaxf(b0, b1);
}

}  // namespace

}  // namespace tracea_amd
