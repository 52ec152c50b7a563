// Host side: from the run-time element type and head dimension of a call to template parameters.
#pragma once
#include <type_traits>
#include "castle_tiles.h"

namespace castle {

// Grid of n workgroups (y of them each) whose kernel asks block_of_many() for its number.  A dispatch counts the threads of a dimension in 32 bits, and those past 2^32 are left out
// without an error: more than 2^21 workgroups stand in x and z, some behind the last one among them.
inline dim3 many_blocks(int64_t n, unsigned y = 1) {
  constexpr int64_t kMost = 1 << 21;
  return n <= kMost ? dim3((unsigned)n, y) : dim3((unsigned)kMost, y, (unsigned)((n + kMost - 1) / kMost));
}

// f(compute type, tensor type): bf16 tensors are converted to fp16 on load (exact inside the fp16 range) and every
// operand produced inside the kernels is fp16, unless bf16_operands asks for bf16 MFMA operands
template <typename F> int by_type(int dtype, bool bf16_operands, F&& f) {
  switch (dtype) {
    case 0: return f(float(), float());
    case 1: return bf16_operands ? f(bf16_t(), bf16_t()) : f(fp16_t(), bf16_t());
    case 2: return f(fp16_t(), fp16_t());
    default: return -1;
  }
}
// f(tensor type)
template <typename F> int by_tensor_type(int dtype, F&& f) {
  switch (dtype) {
    case 0: return f(float());
    case 1: return f(bf16_t());
    case 2: return f(fp16_t());
    default: return -1;
  }
}
template <typename F> int by_type16(int dtype, bool bf16_operands, F&& f) {   // 16-bit tensors only
  if (dtype == 1) return bf16_operands ? f(bf16_t(), bf16_t()) : f(fp16_t(), bf16_t());
  return dtype == 2 ? f(fp16_t(), fp16_t()) : -1;
}
// f(std::integral_constant<int, d>); fp32 kernels exist up to d = 64
template <typename T, typename F> int by_head_dim(int d, F&& f) {
  switch (d) {
    case 16: return f(std::integral_constant<int, 16>());
    case 32: return f(std::integral_constant<int, 32>());
    case 64: return f(std::integral_constant<int, 64>());
    case 128:
      if constexpr (sizeof(T) == 2) return f(std::integral_constant<int, 128>());
      return -2;
    default: return -2;
  }
}

}  // namespace castle
