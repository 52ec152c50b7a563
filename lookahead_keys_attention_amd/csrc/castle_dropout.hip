// Dropout with a residual sum: y = residual + x mask / (1 - p), the mask drawn where it is used, in the backward pass again.
//
// Random numbers: Philox4x32-10 (Salmon, Moraes, Dror, Shaw: Parallel random numbers: as easy as 1, 2, 3, SC 2011).  The key is seed[0], the counter
// (group, seed[1]), all of 64 bits; a group is eight elements of the contiguous tensor, which take the eight 16-bit halves of the
// four words, low half first.  16 bits a number: p is rounded to 1 / 65536, and what stays is divided by what 1 - p then is, so the mean is kept; 32 bits a
// number would double the multiplications, 20 full 32-bit products of a group, which are the only work beside the memory's.
//
// Bound by HBM, one pass: 65536 rows of 2048 bf16 with a residual 144 us (5.6 TB/s), the backward pass without one 83 us (6.5 TB/s).
#include "castle_tiles.h"
#include "castle_dispatch.h"
#include "castle_tokens.h"

namespace castle {
namespace {

struct Words { uint32_t w[4]; };
__device__ __forceinline__ Words philox(uint64_t counter, uint64_t key, uint64_t at) {
  uint32_t a = (uint32_t)counter, b = (uint32_t)(counter >> 32), c = (uint32_t)at, d = (uint32_t)(at >> 32), k0 = (uint32_t)key, k1 = (uint32_t)(key >> 32);
#pragma unroll
  for (int round = 0; round < 10; ++round) {
    const uint64_t p = (uint64_t)0xD2511F53u * a, q = (uint64_t)0xCD9E8D57u * c;
    a = (uint32_t)(q >> 32) ^ b ^ k0;
    c = (uint32_t)(p >> 32) ^ d ^ k1;
    b = (uint32_t)q;
    d = (uint32_t)p;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return {{a, b, c, d}};
}

// A dropped element is zero whatever x holds there: selected, not multiplied.
template <typename T> __device__ __forceinline__ float kept(T x, const Words& r, int e, uint32_t threshold, float scale) {
  const uint32_t u = r.w[e >> 1] >> (e & 1 ? 16 : 0) & 0xffffu;
  return u >= threshold ? (float)x * scale : 0.f;
}

template <typename T, bool RESIDUAL> __global__ __launch_bounds__(kThreads) void dropout_kernel(DropoutArgs a) {
  typedef vec<float, 8> vf;
  const uint64_t key = (uint64_t)a.seed[0], at = (uint64_t)a.seed[1];
  const T *x = static_cast<const T*>(a.x), *res = static_cast<const T*>(a.residual);
  T* y = static_cast<T*>(a.y);
  const int64_t i = block_of_many() * kThreads + threadIdx.x, first = i * 8;
  if (first >= a.n) return;
  if (first + 8 <= a.n) {
    const frag<T> v = *reinterpret_cast<const frag_mem<T>*>(x + first);
    vf s;
    if constexpr (RESIDUAL) s = __builtin_convertvector(*reinterpret_cast<const frag_mem<T>*>(res + first), vf);
    const Words r = philox((uint64_t)i, key, at);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float k = kept<T>(v[e], r, e, a.threshold, a.scale);
      s[e] = RESIDUAL ? s[e] + k : k;
    }
    *reinterpret_cast<frag_mem<T>*>(y + first) = __builtin_convertvector(s, frag<T>);
    return;
  }
  const Words r = philox((uint64_t)i, key, at);
#pragma unroll
  for (int e = 0; e < 8; ++e)
    if (first + e < a.n) {
      const float k = kept<T>(x[first + e], r, e, a.threshold, a.scale);
      y[first + e] = (T)(RESIDUAL ? (float)res[first + e] + k : k);
    }
}

}  // namespace

int launch_dropout(const DropoutArgs& a, int dtype, hipStream_t stream) {
  const int64_t blocks = ((a.n + 7) / 8 + kThreads - 1) / kThreads;
  return by_tensor_type(dtype, [&](auto t) {
    using T = decltype(t);
    if (a.residual != nullptr) hipLaunchKernelGGL((dropout_kernel<T, true>), many_blocks(blocks), dim3(kThreads), 0, stream, a);
    else hipLaunchKernelGGL((dropout_kernel<T, false>), many_blocks(blocks), dim3(kThreads), 0, stream, a);
    return hipGetLastError() == hipSuccess ? 0 : -3;
  });
}

}  // namespace castle
