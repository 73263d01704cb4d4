// Host API of the vocabulary-head losses (see head_loss.cu).
#pragma once
#include <cuda_bf16.h>
#include <cuda_runtime.h>

namespace osb {

constexpr int kHeadRowPad = 256;      // compact row buffers are padded to this many rows
constexpr int kHeadMaxListed = 512;   // listed columns per row

// Everything the forward and backward passes of one call share.  Rows that count are
// numbered 0 .. *count - 1 ("compact" rows); row_of / compact_of translate.  Every row has
// a list of `K` columns, ascending, padded with INT_MAX: the target (K = 1), or the
// teacher's columns with their masses.
struct HeadLossState {
  const __nv_bfloat16* h;      // [R, H] hidden rows, row stride ldh (forward only)
  long long ldh;
  const __nv_bfloat16* w;      // [V, H] head, row stride ldw
  long long ldw;
  int R, H, V, K;
  int rpad;                    // R rounded up to kHeadRowPad
  const float* inv_temp;       // [R] or null
  int divergence;              // 0: cross entropy, 1: divergence from listed teacher logits
  int rest_bucket;             // divergence: the unlisted columns are one more outcome
  float smoothing, z_loss;     // cross entropy
  __nv_bfloat16* hc;           // [rpad, H] compact hidden rows; rows count .. next multiple of 256 are zero
  int* row_of;                 // [rpad] compact row -> row, -1 behind the last
  int* compact_of;             // [R] row -> compact row, -1 for rows that do not count
  int* count;                  // [1]
  int* list_id;                // [R, K]
  float* list_mass;            // [R, K] teacher mass (divergence), unused for cross entropy
  float* list_logit;           // [R, K] student logits of the listed columns
  float* rest_mass;            // [R] teacher mass outside the list (divergence)
  float* all_mass;             // [R] listed and rest mass (divergence): 1 but for a teacher whose list was rounded
  float4* row_stat;            // [R]: lse; then cross entropy: mass of the unlisted columns, factor of q, unused; divergence:
                               // lse of the unlisted columns, factor of their own softmax, factor of q on listed ones
  float* loss;                 // [R]
  int* status;
};

// Index inputs of the two losses.
struct HeadTargets {
  const void* ids;             // [R] or [R, K]
  int ids_i64;
  long long ignore_index;      // cross entropy
  const void* teacher;         // divergence: [R, K] logits
  int teacher_bf16;
  const float* teacher_lse;    // divergence: [R] or null
  unsigned char* active;       // [R] scratch
};

struct HeadStatsScratch {
  float2* part;                // [rpad, tiles] max and sum exp of every vocabulary tile, or of every warp's share
  float* part_sum;             // [rpad, tiles] sum of logits (smoothing > 0) or null
  int tiles;
  char* kept;                  // what the backward pass needs of the logits (HeadKept), or null; `part` lies in it
                               // for many rows
};

// Backward scratch and outputs.
struct HeadGradArgs {
  const float* g;              // [R] upstream gradient
  const char* kept;            // what the forward pass kept of the logits, or null
  float4* row_coef;            // [rpad]
  float* list_grad;            // [R, K]
  __nv_bfloat16* dl;           // [rpad, piece] gradient of one piece of the logits, or [piece, few rows]
  int piece;                   // vocabulary columns a piece (multiple of 256)
  float* dh_part;              // [splits, rpad, H] or null
  int splits;
  __nv_bfloat16* dh;           // [R, H] contiguous or null
  __nv_bfloat16* dw;           // [V, H] contiguous or null
};

// What a forward pass keeps of the logits for a backward pass: of few rows the logits, [V, pitch] fp32; of many their
// exponentials about the maxima of 128 columns, [rpad, pitch] fp16, and behind them those maxima (`part`).
struct HeadKept {
  long long bytes;             // 0: nothing is kept, the logits are computed again
  int pitch;
  long long part_at;           // many rows: where `part` begins
  int tiles;                   // and its row length
};
HeadKept head_loss_kept(int R, int H, int V);
int head_loss_vocab_tiles(int R, int V, bool kept);     // tiles of the statistics scratch
int head_loss_grad_rows(int R);                         // rows (or row pitch) of the logits' gradient
int head_loss_piece(int R, int V);                      // default backward piece
int head_loss_splits(int R, int H, int piece, int V, bool with_dw);   // parts of the hidden gradient's reduction

cudaError_t head_loss_rows_launch(const HeadLossState& s, const HeadTargets& t, cudaStream_t stream);
cudaError_t head_loss_forward_launch(const HeadLossState& s, const HeadStatsScratch& p, cudaStream_t stream);
cudaError_t head_loss_backward_launch(const HeadLossState& s, const HeadGradArgs& g, cudaStream_t stream);

}  // namespace osb
