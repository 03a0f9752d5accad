// Argument blocks and launchers of the operators over a key/value cache in pages: norms of heads with rotary positions, appending, attention.
#pragma once
#include "train.hpp"

namespace tracea_amd {

// Element type of a cache in 8 bits (kernels take the other types' DataType).
constexpr int DT_E4M3 = TRACEA_DTYPE_FLOAT8_E4M3;

// A cache [N, Hk, P, D], D contiguous: strides in bytes.
struct PageView {
  unsigned char *p;
  long long sn, sh, ss;
};
struct ScaleView {  // [N, Hk], strides in elements; p null: a cache of 16 bits
  float *p;
  long long sn, sh;
};
// Page `i` of sequence b: table[b * sb + i], i < M; pages outside 0..N-1 are not there.
struct PageTable {
  const int *p;
  long long sb;
  int M, N, P;
};

// The page of tokens slot * P .. + P - 1 of sequence b, or -1: none.
__host__ __device__ inline int page_of(const PageTable &t, int b, long long slot) {
  if (slot < 0 || slot >= t.M) return -1;
  const int page = t.p[(long long)b * t.sb + slot];
  return page >= 0 && page < t.N ? page : -1;
}

// Norms of heads and rotary positions; positions and pairs as in RotaryArgs (P 0: no positions).
struct QkNormArgs {
  HeadView x[2], out[2], dout[2];  // queries, keys; forward: x -> out, backward: x, dout -> out
  const float *w[2];               // [D] or null (ones)
  float *dw[2];                    // backward: [D] or null
  int H[2];                        // heads; H[1] 0: no keys
  const int *positions;
  long long pos_sb, pos_ss;
  const float *inv_freq;
  int B, S, D, P, axes;
  int first[TRACEA_MAX_ROTARY_AXES];
  int adjacent;
  int vec;     // elements of a piece: 16, 8 or 4 bytes; 0: one by one
  float eps, inv_d;
  int beside;  // lane groups next to each other that take the heads of a token in turn
  int lanes;   // of a lane group, which has a row: a power of two
  int blocks;  // backward: workgroups, which take the tokens in turn
  float *partial;  // backward: [2][blocks][D] sums over a workgroup's rows
};
int launch_qk_norm_forward(const QkNormArgs &a, int dtype, hipStream_t stream);
int launch_qk_norm_backward(const QkNormArgs &a, int dtype, hipStream_t stream);
constexpr int kQkNormMaxDim = 512;
constexpr int kQkNormRuns = 4;  // workgroups a CU of the backward pass, at most

struct CacheAppendArgs {
  HeadView q, q_out, k, v;  // q.p null: no queries
  int Hq, Hk;
  PageView kc, vc;
  ScaleView ks, vs;
  PageTable table;
  const int *starts, *lengths;  // [B]; lengths null: T
  const int *positions;         // null: the token's place in its sequence, one axis
  long long pos_sb, pos_ss;
  const float *inv_freq;
  int B, T, D, P, axes;  // P pairs
  int first[TRACEA_MAX_ROTARY_AXES];
  int adjacent;
  int vec;           // elements of a piece: 8, 4, 2 or 1
  int held;          // rows on 16 bytes, pairs in fours, offsets between the tokens of a page in 31 bits
  int pages;         // that the T tokens of a sequence can touch
  int groups;        // of heads
  int heads, queries;  // key/value and query heads of a group
};
constexpr int kAppendHeads = 64;  // key/value heads of a workgroup, at most
// What the kernel for any sizes works on at once, so that its pieces (up to 512 a row) are counted in 32 bits, whatever pages and heads there
// are: tokens whose sines and cosines fit 32 KB, as many where nothing is turned, and heads of queries.
constexpr int kAppendAngles = 4096, kAppendQueries = 512;
__host__ __device__ inline int append_tokens_at_once(int P) { return P > 0 ? kAppendAngles / P : kAppendAngles; }
int launch_cache_append(const CacheAppendArgs &a, int dtype, hipStream_t stream);

struct AttentionCachedArgs {
  HeadView q, o;
  float *lse;  // null: not wanted
  long long lse_sb, lse_sh, lse_ss;
  PageView k, v;
  ScaleView ks, vs;
  PageTable table;
  unsigned page_magic;  // ceil(2^32 / (P / 16)), 0 for P = 16
  const int *q_len, *k_len;
  int B, Hk, G, Sq, D;
  unsigned g_magic;  // as in AttentionTrainArgs
  float scale_log2;  // magnitude
  int negate, causal;
  int q_vec, o_vec;  // 16-byte pieces
  int rows;        // of a block: 16 or 32 (waves share the keys), 128 (they share tiles of them)
  int row_blocks;  // blocks of rows of a (sequence, key/value head)
  int step, step_log2;  // keys of a workgroup's step
  int workgroups;  // up to 32 rows; 0: one for each block of rows; else the steps of all of them are shared out evenly,
  int shares, apart;  // every problem by itself, in parts of 1 / shares of all steps if these have no more than `apart`
  int twice;       // (of half as many where they have more than this) and if the workgroups are enough for the parts,
  int line;        // or all problems in a line, to so many
  int splits;      // 128 rows: parts of a block's steps
  int *meta;       // [problems][2]: first slot of its parts or -1, their number; null: no problem is cut
  int slots;       // from one part to the next: 2 (up to 32 rows) or 1
  int all_slots;   // of the workspace
  float *part_o, *part_ml;  // [slot][rows][64 or 128], [..][2]
};
constexpr int kCachedStep = 128, kCachedTile = 64;
int launch_attention_cached(const AttentionCachedArgs &a, int dtype, bool e4m3, hipStream_t stream);
int launch_attention_cached_tiles(const AttentionCachedArgs &a, int dtype, bool e4m3, hipStream_t stream);

}  // namespace tracea_amd
