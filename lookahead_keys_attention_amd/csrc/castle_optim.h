// Launchers of castle_optim.hip.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace castle {

constexpr int kTensorsOfLaunch = 64;      // tensors in the arguments of a launch (4 KB)
constexpr int kNormGroups = 2048;         // partial sums of a launch of the norm, at most
constexpr int kScaleBlock = 256;          // elements that share an exponent

struct OptimTensor {
  void* p;              // n elements of the type
  const void* g;
  void *m, *v;          // float, or e4m3 numbers
  int8_t *em, *ev;      // exponents of 256 of them, or nullptr
  int64_t n;
};
// what a launch needs to know of a step, formed on the device by one workgroup in front of it
struct StepNumbers {
  float clip, rate, root, keep;   // factor of the gradients, lr / (1 - b1^t), 1 / sqrt(1 - b2^t), 1 - lr wd
  uint32_t step, unused[3];
};
struct StepOptions {
  double lr, b1, b2, eps, weight_decay, max_norm;   // max_norm < 0: gradients as they are
  const float* lr_device;     // or nullptr
  int64_t* step;              // steps taken; one more behind the call
  const int64_t* seed;        // nullptr: nearest
};
int64_t optim_workspace(int count);
int launch_grad_norm(const OptimTensor* tensors, int count, float* norm, int dtype, void* workspace, hipStream_t stream);
// norm: nullptr, or what the gradients are clipped by; clip_here: it is formed here first (and written to `norm`)
int launch_adamw(const OptimTensor* tensors, int count, const StepOptions& o, float* norm, bool clip_here, int dtype, void* workspace, hipStream_t stream);

}  // namespace castle
