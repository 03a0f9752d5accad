// Argument blocks and launchers of the kernels for training: attention with row statistics and its backward pass,
// rotary positions, and the norm / gate / residual sum between two blocks.
#pragma once
#include "common.hpp"

namespace tracea_amd {

// One tensor [B, heads, rows, D] with D contiguous: element strides of batch, head and row.
struct HeadView {
  void *p;
  long long sb, sh, ss;
};

// Attention with Hq = G * Hk heads.  The G query heads that share a key/value head are worked on as one matrix of
// packed rows: row r of (b, hk) is query r / G of head hk * G + r % G, so that a tile of rows is a run of queries (what a
// causal mask cuts) with all heads of the group, K and V are read once for the group and sums over the heads of a group are
// sums over rows.
struct AttentionTrainArgs {
  HeadView q, k, v, o, d_o, dq, dk, dv;
  float *lse;  // [B, Hq, Sq] by these strides
  long long lse_sb, lse_sh, lse_ss;
  const int *q_len, *k_len;  // [B] or null
  int B, Hk, G, Sq, Sk, D;
  unsigned g_magic;   // ceil(2^32 / G) (G > 1): r / G = umulhi(r, g_magic) while G * G * Sq < 2^32
  float scale, scale_log2;  // magnitudes; negate: the caller's scale is below zero
  int negate, causal;
  int order;  // of the workgroups: 0 runs of heads, 1 heaviest blocks first, 2 those going round the XCDs
  // backward: per packed row -lse * log2(e) (-inf: nothing visible) and -(dO . O), [B * Hk][rows_pad] each
  float *neg_lse2, *neg_delta;
  int rows_pad;  // G * Sq up to a multiple of 64
  int block;       // columns (packed rows, keys) of a workgroup: 128; 64, two waves on 32 columns; forward only: 32, two waves on 16 rows
  int row_splits;  // parts of the rows for dK and dV, each with a workgroup of its own
  float *part_dkv; // [row_splits][B * Hk][Sk][dK, dV][width], row_splits > 1
  // f16 only: largest squared row norms of dO and V, [B * Hk][norm_blocks] (64 rows of dO or 64 keys of V each)
  float *norms;
  int norm_blocks;
  // forward over a split key axis: partial results (o in fp32 unnormalised, running maximum and sum per row)
  int splits, steps_per_split;  // steps: 64 keys, or 128 with two waves on the same rows
  float *part_o, *part_ml;
};

// Rotary positions: one or two tensors [B, heads, S, D] turned by the same angles.
struct RotaryArgs {
  HeadView q, k, q_out, k_out;
  int Hq, Hk;  // Hk 0: no second tensor
  const int *positions;
  long long pos_sb, pos_ss;  // pos_sb 0: one set for the batch
  const float *inv_freq;
  int B, S, D, P, axes;
  int first[TRACEA_MAX_ROTARY_AXES];  // first pair of the axis
  int adjacent, inverse;
  int vec;  // 16-byte pieces: columns, strides and bases allow it
  int heads_per_group, beside;  // a workgroup has a group of heads of its tokens; `beside` threads next to each other take them in turn
};
int launch_rotary(const RotaryArgs &a, int dtype, hipStream_t stream);

// The sum between two blocks and the norms on both sides of it.  Rows [B, T, C] by (batch, row) strides, C contiguous.
struct RowView {
  void *p;
  long long sb, ss;
};
struct NormArgs {
  RowView x, h, x_out, y;              // forward; backward reads h, x_out
  RowView dx_out, dy, dx, dh;
  const float *w_post, *gate, *w_pre;  // gate [G, C]; absent: 1 (null), together with the tensors they belong to
  float *dw_post, *dgate, *dw_pre;     // null: not wanted
  long long gate_sb;                   // 0: one for the batch
  int B, T, C;
  float eps, scale;
  int vec;  // 16-byte pieces
  int chunks, rows_per_chunk;  // workgroups per batch entry and the rows of each
  float *partial;              // backward: [2][B * chunks][C] column sums of dt * h^ and dy * x^
};
int launch_norm_forward(const NormArgs &a, int dtype, hipStream_t stream);
int launch_norm_backward(const NormArgs &a, int dtype, hipStream_t stream);
// Workgroups per batch entry for T rows of C channels.
int norm_chunks(int B, int T, int C, int cus, bool backward);
constexpr int kNormMaxChannels = 8192;

int launch_attention_train_forward(const AttentionTrainArgs &a, int dtype, hipStream_t stream);
int launch_attention_train_backward(const AttentionTrainArgs &a, int dtype, hipStream_t stream);

}  // namespace tracea_amd
