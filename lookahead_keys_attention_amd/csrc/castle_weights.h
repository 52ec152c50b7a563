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
struct WeightsPlan { int whole, rest, ranges, steps; float cost; };   // tiles taken whole, the others, ranges of each of those and steps of a range; cost: us

WeightsPlan weights_plan(int R, int M0, int N0, int M1, int N1);
int64_t weights_workspace(const WeightsPlan& p);
int launch_weights(const WeightProduct& first, const WeightProduct& second, int R, const WeightsPlan& p, int dtype, float* workspace, hipStream_t stream);

}  // namespace castle
