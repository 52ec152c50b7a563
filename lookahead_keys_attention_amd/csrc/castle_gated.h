// Launchers of castle_gated.hip: u = x w_in^T, (g, v) the halves of its columns, h = act(g) v, y = h w_out^T.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace castle {

enum { kSilu = 0, kGeluGate = 1 };
struct GatedArgs {
  const void *x, *w_in, *w_out;   // [R][ld_x], [2 F][ld_in], [D][ld_out]
  int64_t ld_x, ld_in, ld_out;
  int R, D, F, act;
};
int64_t gated_state(int R, int D, int F, int dtype);
int64_t gated_workspace(int R, int D, int F, int dtype, bool keeps);
int64_t gated_bwd_workspace(int R, int D, int F, int dtype, int gradients);
int launch_gated(const GatedArgs& a, void* y, void* state, int dtype, void* workspace, hipStream_t stream);
// gradients that are nullptr are not formed
int launch_gated_bwd(const GatedArgs& a, const void* dy, const void* state, void* dx, void* dw_in, void* dw_out, int dtype, void* workspace, hipStream_t stream);

}  // namespace castle
