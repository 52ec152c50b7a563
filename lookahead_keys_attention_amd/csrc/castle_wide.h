// Operands of products whose tiles belong to workgroups of eight waves: straight from memory to LDS, 64 steps of the contraction at a time.
#pragma once
#include "castle_tiles.h"
#include "castle_waves.h"

namespace castle {

constexpr int kWideK = 64, kWideThreads = 512;
// FREE rows or columns; KC: the operand is contraction-contiguous, else stored [contraction][free].
// 16-byte pieces go to LDS in the order of the lanes, so rows cannot be padded: a piece takes another place in its row instead, such that
// the lanes of a read spread over all banks (contraction-contiguous: piece p of row r at p ^ (r / 2 % 8); else the pieces of row k
// at p ^ 4 (k % 4)).
template <typename T, bool KC, int FREE> struct WideOperand {
  static constexpr int N = FREE / 64;   // loads of a wave
  const T* at;
  uint32_t off[N];   // bytes
  int left;          // rows or columns of the tile that are there
  __device__ __forceinline__ void start(const T* p, int64_t ld, int free0, int free_end, int k0) {
    at = KC ? p + free0 * ld + k0 : p + k0 * ld + free0;
    left = free_end - free0;
    place((int)ld, kWideK);
  }
  // steps: what is left of the contraction; behind its end the last row is read again (or load_end)
  __device__ __forceinline__ void place(int ld, int steps) {
    const int lane = lane_id(), first = wave_id() * N;
#pragma unroll
    for (int q = 0; q < N; ++q) {
      if constexpr (KC) {
        const int row = 8 * (first + q) + (lane >> 3), piece = (lane & 7) ^ (row >> 1 & 7);
        off[q] = 2 * (uint32_t)(ld * min(row, left - 1) + 8 * piece);
      } else {
        constexpr int PIECES = FREE / 8, ROWS = 64 / PIECES;
        const int k = ROWS * (first + q) + lane / PIECES, piece = lane % PIECES ^ 4 * (k & 3);
        off[q] = 2 * (uint32_t)(min(k, steps - 1) * ld + (8 * piece < left ? 8 * piece : 0));
      }
    }
  }
  __device__ __forceinline__ void load(int64_t ld, uint32_t lds) {
#pragma unroll
    for (int q = 0; q < N; ++q) load_to_lds(at, off[q], lds + 1024 * (wave_id() * N + q));
    at += KC ? kWideK : kWideK * ld;
  }
  // The last step of a contraction, `steps` of it left: the pieces behind its end are those 16 bytes of zeros.  (Read again, whatever is not finite there would meet the zeros of
  // the other operand's rows.)
  __device__ __forceinline__ void load_end(int steps, const T* zeros, uint32_t lds) {
    const int lane = lane_id(), first = wave_id() * N;
#pragma unroll
    for (int q = 0; q < N; ++q) {
      bool there;
      if constexpr (KC) {
        const int row = 8 * (first + q) + (lane >> 3), piece = (lane & 7) ^ (row >> 1 & 7);
        there = 8 * piece < steps;
      } else {
        constexpr int PIECES = FREE / 8, ROWS = 64 / PIECES;
        there = ROWS * (first + q) + lane / PIECES < steps;
      }
      load_to_lds_from(there ? reinterpret_cast<const unsigned char*>(at) + off[q] : reinterpret_cast<const unsigned char*>(zeros), lds + 1024 * (first + q));
    }
  }
  // operand fragments of the wave's 32 W columns from free0, 16 contraction steps from 16 s
  template <int W> static __device__ __forceinline__ void read(const T* lds, frag<T> (&f)[W], int free0, int s, int c, int g) {
    if constexpr (KC) {
      const T* p = lds + (free0 + c) * kWideK + 8 * ((2 * s + g) ^ (c >> 1 & 7));
#pragma unroll
      for (int i = 0; i < W; ++i) f[i] = *reinterpret_cast<const frag<T>*>(p + 32 * kWideK * i);
    } else {
      const int lp = c & 15, k = 16 * s + 8 * g + (lp >> 2);
#pragma unroll
      for (int i = 0; i < W; ++i) {
        const T* p = lds + k * FREE + 32 * ((free0 / 32 + i) ^ (lp >> 2)) + 16 * (c >> 4) + 4 * (lp & 3);
        const vec<T, 4> lo = lds_tr4<T>(p), hi = lds_tr4<T>(p + 4 * FREE);
#pragma unroll
        for (int e = 0; e < 4; ++e) { f[i][e] = lo[e]; f[i][4 + e] = hi[e]; }
      }
    }
  }
};

}  // namespace castle
