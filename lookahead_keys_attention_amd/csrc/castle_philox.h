// Philox4x32-10 (Salmon, Moraes, Dror, Shaw: Parallel random numbers: as easy as 1, 2, 3, SC 2011).
#pragma once
#include <stdint.h>
#include <hip/hip_runtime.h>

namespace castle {

struct Words { uint32_t w[4]; };
__device__ __forceinline__ uint32_t xor3(uint32_t a, uint32_t b, uint32_t c) { return __builtin_amdgcn_bitop3_b32(a, b, c, 0x96); }
__device__ __forceinline__ Words philox(uint64_t counter, uint64_t key, uint64_t at) {
  uint32_t a = (uint32_t)counter, b = (uint32_t)(counter >> 32), c = (uint32_t)at, d = (uint32_t)(at >> 32), k0 = (uint32_t)key, k1 = (uint32_t)(key >> 32);
#pragma unroll
  for (int round = 0; round < 10; ++round) {
    const uint64_t p = (uint64_t)0xD2511F53u * a, q = (uint64_t)0xCD9E8D57u * c;
    a = xor3((uint32_t)(q >> 32), b, k0);
    c = xor3((uint32_t)(p >> 32), d, k1);
    b = (uint32_t)q;
    d = (uint32_t)p;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return {{a, b, c, d}};
}
// one of the eight 16-bit halves, low half first
__device__ __forceinline__ uint32_t half_of(const Words& r, int e) { return r.w[e >> 1] >> (e & 1 ? 16 : 0) & 0xffffu; }

}  // namespace castle
