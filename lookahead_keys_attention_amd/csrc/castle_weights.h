// Launcher of castle_weights.hip.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace castle {

// c [M][N] = a^T b, a [R][lda], b [R][ldb]
struct WeightProduct {
  const void *a, *b;
  void* c;
  int M, N;
  int64_t lda, ldb;
};
struct WeightsPlan {   // tiles taken whole, the others, ranges of each of those and steps of a range; cost: us
  int whole, rest, ranges, steps;
  float cost;
  int x_groups, longs, long_steps;   // with the input gradient: workgroups of an XCD that have a tile of it; of the ranges the first `longs` have long_steps, the others `steps`
};

WeightsPlan weights_plan(int R, int M0, int N0, int M1, int N1);
WeightsPlan gradients_plan(int R, int M0, int N0, int M1, int N1, int M, int N, int K);
int64_t weights_workspace(const WeightsPlan& p);
// x: nullptr, or the input gradient, of `K` (gradients_plan)
int launch_weights(const WeightProduct& first, const WeightProduct& second, const WeightProduct* x, int K, int R, const WeightsPlan& p, int dtype, float* workspace, hipStream_t stream);

}  // namespace castle
