// What stands between the two products of a gated feed-forward block.
#pragma once
#include "castle_gated.h"
#include "castle_gelu.h"

namespace castle {

// act(g) and its derivative
template <typename T, int ACT> struct Gate {
  float act, slope;
  __device__ __forceinline__ explicit Gate(float g) {
    if constexpr (ACT == kSilu) {
      const float s = sizeof(T) == 4 ? 1.f / (1.f + expf(-g)) : sigmoid_l2(g * kLog2e);
      act = g * s;
      slope = __builtin_fmaf(act, 1.f - s, s);
    } else {
      const Normal<T> n(g);
      act = g * n.cdf;
      slope = __builtin_fmaf(g * 0.3989422804f, n.e, n.cdf);
    }
  }
};

}  // namespace castle
