// Launchers of castle_dropout.hip and castle_embedding.hip.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace castle {

struct DropoutArgs {
  const void *x, *residual;   // n elements; residual may be nullptr
  void* y;
  const int64_t* seed;        // two numbers in device memory
  int64_t n;
  uint32_t threshold;         // of 65536: an element stays where its 16 bits are at least this
  float scale;
};
int launch_dropout(const DropoutArgs& a, int dtype, hipStream_t stream);

// token r: index[(r / n) * index_ld + r % n]
struct TokenRows {
  const int64_t* index;
  int64_t rows, n, index_ld;
};
struct EmbeddingArgs {
  TokenRows tokens;
  const void* table;   // [V][ld]
  int64_t ld;
  void* y;             // [rows][D]
  int V, D;
  float scale;
};
int launch_embedding(const EmbeddingArgs& a, int dtype, hipStream_t stream);

// Gradient of the embedding by sorted tokens: sizes of what lies in the workspace, in this order
struct SortedGradPlan {
  int passes, bits;        // of a digit
  bool together;           // the sort in one workgroup
  int groups;              // workgroups of a sorting pass
  int64_t wave_tokens;     // tokens of a wave of them
  int rows_per_group;      // vocabulary rows of a workgroup of the sums
  int64_t counts, keys, places, parts, ranges, total;   // bytes
};
struct SortedGradArgs {
  TokenRows tokens;
  const void* dy;      // [rows][D]
  void* dw;            // [V][D]
  int V, D, padding;   // tokens equal to `padding` (-1: none) and those outside 0 .. V - 1 have no part in it
  float scale;
  SortedGradPlan plan;
  void* workspace;
};
SortedGradPlan sorted_grad_plan(int64_t rows, int V, int D);
int launch_sorted_grad(const SortedGradArgs& a, int dtype, hipStream_t stream);

}  // namespace castle
