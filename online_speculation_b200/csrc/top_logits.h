// Host API of the top-logits kernel (see top_logits.cu).
#pragma once
#include <cuda_runtime.h>

namespace osb {

constexpr int kTopLogitsMax = 512;

struct TopLogitsArgs {
  const void* logits;        // [R, V] fp32 or bf16, row stride ld, unit column stride
  int bf16;
  long long ld;
  int R, V, k;
  const float* inv_temp;     // [R] or null
  float* values;             // [R, k]
  int* ids;                  // [R, k]
  float* lse;                // [R]
  int splits;                // column ranges per row
  unsigned long long* keys;  // [R, splits, k] when splits > 1
  float2* part;              // [R, splits] when splits > 1
};

int top_logits_splits(int R, int V, int k);
cudaError_t top_logits_launch(const TopLogitsArgs& a, cudaStream_t stream);

}  // namespace osb
