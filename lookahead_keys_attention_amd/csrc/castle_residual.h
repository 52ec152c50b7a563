// Launchers of castle_residual.hip.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace castle {

// rows of D elements, contiguous, of any alignment; what is nullptr is not there
struct ResidualArgs {
  const void *x, *residual, *w, *scale, *next_w;   // w, scale, next_w: [D]
  const void* gate;      // [rows / span][D]: row r has that of r / span
  int64_t rows, span;
  int D;
  float eps;
  float *rstd, *next_rstd;   // [rows], for the backward pass
  void *y, *h;
};
struct ResidualBwdArgs {
  ResidualArgs f;            // (y and h are not read)
  const void *dy, *dh;       // gradients of y and of h
  void *dx, *dresidual, *dgate;
  void *dw, *dscale, *dnext;
};
constexpr int kResidualMaxWidth = 8192;
int64_t residual_bwd_workspace(const ResidualBwdArgs& a);
int launch_residual(const ResidualArgs& a, int dtype, hipStream_t stream);
int launch_residual_bwd(const ResidualBwdArgs& a, int dtype, void* workspace, hipStream_t stream);

}  // namespace castle
