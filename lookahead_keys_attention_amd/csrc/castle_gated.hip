// Gated feed-forward block:  u = x w_in^T, (g, v) the halves of u's columns, h = act(g) v, y = h w_out^T
//   dh = dy w_out     dg = dh v act'(g)     dv = dh act(g)     dx = [dg dv] w_in     dw_in = [dg dv]^T x     dw_out = dy^T h
#include "castle_tiles.h"
#include "castle_dispatch.h"
#include "castle_gate.h"
#include "castle_gemm.h"
#include "castle_rows.h"
#include "castle_weights.h"
#include "castle_wide.h"
#include <algorithm>

namespace castle {
namespace {

typedef vec<float, 8> vf;

// ---- fp32: u in memory, the gate on the store of its product (castle_gemm32.hip) or, where that goes in ranges, by itself -------
__device__ __forceinline__ vf load8(const float* p) { return *reinterpret_cast<const frag_mem<float>*>(p); }
__device__ __forceinline__ void store8(float* p, vf v) { *reinterpret_cast<frag_mem<float>*>(p) = v; }
// h of u = [R][2 F]
template <int ACT> __global__ __launch_bounds__(kThreads) void gate_kernel(const float* u, int64_t n, int F, float* h) {
  const int64_t i = (block_of_many() * kThreads + threadIdx.x) * 8, row = i / F, at = row * 2 * F + i - row * F;
  if (i >= n) return;
  const vf g = load8(u + at), v = load8(u + at + F);
  vf y;
#pragma unroll
  for (int e = 0; e < 8; ++e) y[e] = Gate<float, ACT>(g[e]).act * v[e];
  store8(h + i, y);
}
// [dg dv] of dh and u, and h; dh or h may be nullptr
template <int ACT> __global__ __launch_bounds__(kThreads) void gate_bwd_kernel(const float* u, const float* dh, int64_t n, int F, float* du, float* h) {
  const int64_t i = (block_of_many() * kThreads + threadIdx.x) * 8, row = i / F, at = row * 2 * F + i - row * F;
  if (i >= n) return;
  const vf g = load8(u + at), v = load8(u + at + F), d = dh != nullptr ? load8(dh + i) : vf{};
  vf dg, dv, y;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const Gate<float, ACT> a(g[e]);
    dg[e] = d[e] * (v[e] * a.slope);
    dv[e] = d[e] * a.act;
    y[e] = a.act * v[e];
  }
  if (dh != nullptr) {
    store8(du + at, dg);
    store8(du + at + F, dv);
  }
  if (h != nullptr) store8(h + i, y);
}

// ---- 16-bit types: the gate inside the products ---------------------------------------------------------------------
// Tiles of BM rows by 128 hidden columns.  Forward: of a step of the contraction both halves of w_in lie in LDS, 32 of its rows and 32 of the other half in turn, so that a wave holds g and v of the
// same elements in its accumulators and u never leaves them: h goes to memory and, for the backward pass, a = act(g) and b = v act'(g), in the order of the registers.  Backward: the tile of dh = dy w_out
// meets a and b in the same order, and [dg dv] = [dh b, dh a] goes to memory.  a and b keep 24 of their 32 bits (one part of 16 and one of 8): as 16-bit numbers each would be
// rounded twice on the way to dg and dv, and the gradients were twice as far from the formula as rounded once; with h and [dg dv] alone rounded it is 1.4 times.
enum { kForward = 0, kForwardKeep = 1, kBackward = 2 };
struct GatedProductArgs {
  const void *a, *b;       // x and w_in; dy and w_out
  int64_t lda, ldb;
  int R, F, K;             // K: of the contraction
  void* out;               // h [R][F]; [dg dv] [R][2 F]
  unsigned char* planes;   // a and b: [tile][wave][piece of 32 x 32] of kPlaneBytes
};
constexpr int kTileF = 128;             // hidden columns of a tile
constexpr int kPlaneBytes = 6 * 1024;   // 16 numbers a lane of a and of b: 32 bytes of each of their first parts, 16 of the others
template <int MODE, int BM> struct GatedShape {
  static constexpr int BN = MODE == kBackward ? kTileF : 2 * kTileF;
  static constexpr int WM = BM == 256 ? 4 : 2, WN = 8 / WM, FM = BM / 32 / WM, FN = BN / 32 / WN, FH = kTileF / 32 / WN;   // pieces of a wave: rows, columns of the product, hidden columns
  static constexpr int kLoadsA = BM / 64, kLoads = kLoadsA + BN / 64, kBytesA = kLoadsA * 8 * 1024, kStage = kLoads * 8 * 1024;
  static constexpr int kTurn = 2048, kFit = (kMaxLds - 8 * kTurn) / kStage, kStages = kFit < 3 ? kFit : 3, kLds = kStages * kStage + 8 * kTurn;
  static constexpr int kStores = FM * FH * (MODE == kForward ? 2 : MODE == kForwardKeep ? 8 : 4);   // of a wave and tile
  static_assert(kStages >= 2 && FM >= 1 && FH >= 1, "");
};
__device__ const uint32_t castle_gated_zeros[4] __attribute__((aligned(16))) = {0, 0, 0, 0};
extern __shared__ __attribute__((aligned(16))) unsigned char castle_gated_lds[];

// PAIRS: rows 64 k .. 64 k + 31 of the tile are rows 32 k .. of the first half of the matrix, the next 32 the same of its second half, `half` elements further on
template <typename T, bool KC, int FREE, bool PAIRS> struct GatedOperand : WideOperand<T, KC, FREE> {
  typedef WideOperand<T, KC, FREE> W;
  static constexpr int N = W::N;
  __device__ __forceinline__ void start(const T* p, int64_t ld, int free0, int free_end, uint32_t half) {
    W::start(p, ld, free0, free_end, 0);
    if constexpr (PAIRS) {
      const int lane = lane_id(), first = wave_id() * N;
#pragma unroll
      for (int q = 0; q < N; ++q) {
        const int row = 8 * (first + q) + (lane >> 3), piece = (lane & 7) ^ (row >> 1 & 7), there = min(row / 64 * 32 + row % 32, W::left - 1);
        W::off[q] = 2 * ((uint32_t)((int)ld * there + 8 * piece) + (row & 32 ? half : 0u));
      }
    }
  }
  __device__ __forceinline__ void load_end(int steps, uint32_t lds) { W::load_end(steps, reinterpret_cast<const T*>(castle_gated_zeros), lds); }
};

// x as a number of 32 bits, whoever reads it: a product that is rounded to 16 bits in the same instruction would not be the one whose rest is taken
__device__ __forceinline__ void in_32_bits(float& x) { asm("" : "+v"(x)); }
__device__ __forceinline__ void in_32_bits(vec<float, 16>& x) {
#pragma unroll
  for (int r = 0; r < 16; ++r) {
    float e = x[r];
    in_32_bits(e);
    x[r] = e;
  }
}
// what x loses when it is rounded to T; of what becomes infinite nothing
template <typename T> __device__ __forceinline__ float rest(float x) {
  const float r = (float)(T)x;
  return __builtin_fabsf(r) == __builtin_inff() ? 0.f : x - r;
}
template <typename T> __device__ __forceinline__ vec<float, 16> rest(const vec<float, 16>& x) {
  vec<float, 16> y;
#pragma unroll
  for (int r = 0; r < 16; ++r) y[r] = rest<T>((float)x[r]);
  return y;
}
typedef vec<uint32_t, 4> u4;
// sixteen numbers of a lane as their upper 24 bits: [0], [1] upper halves, [2] the bytes behind them
__device__ __forceinline__ void to_parts(const vec<float, 16>& x, u4 (&p)[3]) {
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    const uint32_t lo = __builtin_bit_cast(uint32_t, (float)x[2 * k]), hi = __builtin_bit_cast(uint32_t, (float)x[2 * k + 1]);
    p[k / 4][k % 4] = __builtin_amdgcn_perm(hi, lo, 0x07060302);
    if (k % 2 == 0) {
      const uint32_t lo2 = __builtin_bit_cast(uint32_t, (float)x[2 * k + 2]), hi2 = __builtin_bit_cast(uint32_t, (float)x[2 * k + 3]);
      const uint32_t first = __builtin_amdgcn_perm(hi, lo, 0x0c0c0501), second = __builtin_amdgcn_perm(hi2, lo2, 0x0c0c0501);
      p[2][k / 2] = first | second << 16;
    }
  }
}
__device__ __forceinline__ vec<float, 16> from_parts(const u4& p0, const u4& p1, const u4& p2) {
  vec<float, 16> x;
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    const uint32_t upper = k < 4 ? p0[k % 4] : p1[k % 4], lower = p2[k / 2];   // byte 1 of the number from byte k % 2 * 2 (+ 1) of `lower`
    x[2 * k] = __builtin_bit_cast(float, __builtin_amdgcn_perm(upper, lower, k % 2 ? 0x0504020c : 0x0504000c));
    x[2 * k + 1] = __builtin_bit_cast(float, __builtin_amdgcn_perm(upper, lower, k % 2 ? 0x0706030c : 0x0706010c));
  }
  return x;
}

// The frame is that of gemm_wide_kernel (castle_gemm.hip): eight waves, one workgroup to a CU, steps of 64 of the contraction straight from memory to LDS into two or three buffers, requested over the
// end of a tile.  END: the contraction ends inside a step.  LOW: what the rounding of h and of [dg dv] leaves is kept too, in as many rows behind them.
template <typename T, int MODE, int ACT, int BM, bool END, bool LOW> __global__ __launch_bounds__(kWideThreads, 2) void gated_product_kernel(GatedProductArgs a) {
  typedef GatedShape<MODE, BM> S;
  typedef GatedOperand<T, true, BM, false> OpA;
  typedef GatedOperand<T, MODE != kBackward, S::BN, MODE != kBackward> OpB;
  typedef vec<T, 8> vt;
  typedef vec<float, 16> v16;
  const int lane = lane_id(), wave = wave_id(), c = lane & 31, g = lane >> 5;
  // tiles in the order of an XCD's L2: all rows of a band of columns, then those of the next; XCD x takes the x-th eighth
  constexpr int kBand = 2048 / S::BN;
  const int tiles_m = (a.R + BM - 1) / BM, tiles_n = (a.F + kTileF - 1) / kTileF, tiles = tiles_m * tiles_n;
  auto place = [&](int t, int& m, int& n) __attribute__((always_inline)) {
    const int band = t / (tiles_m * kBand), rest = t - band * tiles_m * kBand, width = min(kBand, tiles_n - band * kBand);
    m = rest / width;
    n = band * kBand + rest % width;
  };
  const int share = (tiles + 7) / 8, first = blockIdx.x % 8 * share, last = min(tiles, first + share), stride = gridDim.x / 8;
  const int wm = wave / S::WN * 32 * S::FM, wn = wave % S::WN * 32 * S::FN, wh = wave % S::WN * 32 * S::FH;
  const int steps = (a.K + kWideK - 1) / kWideK;
  int tile = first + blockIdx.x / 8;
  if (tile >= last) return;
  const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) unsigned char*)castle_gated_lds, half = (uint32_t)a.F * (uint32_t)a.ldb;
  // the step that is requested next runs ahead of the one that is multiplied, into the next tile
  OpA ra;
  OpB rb;
  int next_tile = tile, next_step = 0, ahead = 0;   // ahead: steps requested and not waited for
  auto start = [&]() __attribute__((always_inline)) {
    int m, n;
    place(next_tile, m, n);
    ra.start(static_cast<const T*>(a.a), a.lda, m * BM, a.R, 0);
    rb.start(static_cast<const T*>(a.b), a.ldb, n * kTileF, a.F, half);
  };
  auto request = [&](int buffer) __attribute__((always_inline)) {
    if (next_tile >= last) return;
    ++ahead;
    if (END && next_step == steps - 1) {
      const int left = a.K - next_step * kWideK;
      ra.load_end(left, lds0 + buffer);
      rb.load_end(left, lds0 + buffer + S::kBytesA);
    } else {
      ra.load(a.lda, lds0 + buffer);
      rb.load(a.ldb, lds0 + buffer + S::kBytesA);
    }
    if (++next_step == steps) {
      next_step = 0;
      next_tile += stride;
      if (next_tile < last) start();
    }
  };
  start();
  request(0);
  request(S::kStage);
  if constexpr (S::kStages == 3) request(2 * S::kStage);
  // The step behind the current one is in LDS, from every wave, and all have read the current one.  Waits are for all but the last so many requests; the stores of a tile inside the output come
  // behind those and are not waited for (`stored`).
  bool stored = false;
  auto arrive = [&]() __attribute__((always_inline)) {
    auto wait = [&](auto n) __attribute__((always_inline)) {
      asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(decltype(n)::value < 63 ? decltype(n)::value : 63) : "memory");
    };
    const int newer = ahead - 1;   // steps
    if (newer > 1) {
      if (stored) wait(std::integral_constant<int, 2 * S::kLoads + S::kStores>());
      else wait(std::integral_constant<int, 2 * S::kLoads>());
    } else if (newer == 1) {
      if (stored) wait(std::integral_constant<int, S::kLoads + S::kStores>());
      else wait(std::integral_constant<int, S::kLoads>());
    } else {
      if (stored) wait(std::integral_constant<int, S::kStores>());
      else wait(std::integral_constant<int, 0>());
    }
    stored = false;
    --ahead;
  };
  int buffer = 0;
  frag<T> fa[2][S::FM], fb[2][S::FN];
  auto read = [&](int slot, int s) __attribute__((always_inline)) {
    OpA::read(reinterpret_cast<const T*>(castle_gated_lds + buffer), fa[slot], wm, s, c, g);
    OpB::read(reinterpret_cast<const T*>(castle_gated_lds + buffer + S::kBytesA), fb[slot], wn, s, c, g);
    __builtin_amdgcn_sched_barrier(0);   // these reads, then the products of the fragments before
  };
  T* const turn = reinterpret_cast<T*>(castle_gated_lds + S::kStages * S::kStage + wave * S::kTurn);
  arrive();
  while (tile < last) {
    int tm, tn;
    place(tile, tm, tn);
    const int m0 = tm * BM, n0 = tn * kTileF;
    const bool inside = m0 + BM <= a.R && n0 + kTileF <= a.F;
    u4* const planes = reinterpret_cast<u4*>(a.planes + (((int64_t)tm * tiles_n + tn) * 8 + wave) * (S::FM * S::FH * kPlaneBytes)) + lane;
    // (backward: requested before the tile's products, which hide them)
    u4 kept[MODE == kBackward ? S::FM * S::FH : 1][6];
    if constexpr (MODE == kBackward) {
#pragma unroll
      for (int p = 0; p < S::FM * S::FH; ++p)
#pragma unroll
        for (int k = 0; k < 6; ++k) kept[p][k] = __builtin_nontemporal_load(planes + (p * 6 + k) * 64);
    }
    read(0, 0);
    int done = 0;   // buffer of the step that ends
    acc_t acc[S::FM][S::FN];   // [columns, m lanes]
#pragma unroll
    for (int i = 0; i < S::FM; ++i)
#pragma unroll
      for (int j = 0; j < S::FN; ++j) zero(acc[i][j]);
    auto multiply = [&](int slot) __attribute__((always_inline)) {
#pragma unroll
      for (int i = 0; i < S::FM; ++i)
#pragma unroll
        for (int j = 0; j < S::FN; ++j) mma(acc[i][j], fb[slot][j], fa[slot][i]);
    };
    for (int it = 0; it < steps; ++it) {
#pragma unroll
      for (int s = 0; s < kWideK / 16 - 1; ++s) {
        read(1 - s % 2, s + 1);
        multiply(s % 2);
      }
      arrive();
      done = buffer;
      buffer = buffer == (S::kStages - 1) * S::kStage ? 0 : buffer + S::kStage;
      if (it + 1 < steps) request(done);
      read(0, 0);   // (behind the last step: for nothing)
      multiply(1);
    }
    asm volatile("s_nop 15\n\ts_nop 3" ::: "memory");   // the loop may end right behind a product
    __builtin_amdgcn_sched_barrier(0);
    request(done);
    tile += stride;
    // 32 x 32 numbers to whole rows, 64 bytes of each, through the wave's own place in LDS (piece p of row r at p ^ (r / 4 % 4))
    auto to_rows = [&](const v16& z, T* out, int64_t ld, int m, int n) __attribute__((always_inline)) {
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
#pragma unroll
      for (int q = 0; q < 4; ++q) st4<T>(turn + c * 32 + 8 * (q ^ (c >> 2 & 3)) + 4 * g, pack4<T>(z, q));
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const int row = 16 * k + (lane >> 2), piece = lane & 3;
        const vt v = *reinterpret_cast<const vt*>(turn + row * 32 + 8 * (piece ^ (row >> 2 & 3)));
        if (m + row < a.R && n + 8 * piece < a.F) *reinterpret_cast<vt*>(out + (m + row) * ld + n + 8 * piece) = v;
      }
    };
#pragma unroll
    for (int i = 0; i < S::FM; ++i)
#pragma unroll
      for (int j = 0; j < S::FH; ++j) {
        const int m = m0 + wm + 32 * i, n = n0 + wh + 32 * j;
        v16 x, y;
        if constexpr (MODE == kBackward) {
          const u4(&p)[6] = kept[i * S::FH + j];
          x = from_parts(p[0], p[1], p[2]) * acc[i][j];   // dv
          y = from_parts(p[3], p[4], p[5]) * acc[i][j];   // dg
          T* out = static_cast<T*>(a.out);
          if constexpr (LOW) {
            in_32_bits(x);
            in_32_bits(y);
          }
          to_rows(y, out, 2 * (int64_t)a.F, m, n);
          to_rows(x, out + a.F, 2 * (int64_t)a.F, m, n);
          if constexpr (LOW) {
            out += (int64_t)a.R * 2 * a.F;
            to_rows(rest<T>(y), out, 2 * (int64_t)a.F, m, n);
            to_rows(rest<T>(x), out + a.F, 2 * (int64_t)a.F, m, n);
          }
        } else {
          v16 h;
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const Gate<T, ACT> gate(acc[i][2 * j][r]);
            x[r] = gate.act;
            y[r] = acc[i][2 * j + 1][r] * gate.slope;
            h[r] = acc[i][2 * j + 1][r] * gate.act;
          }
          if constexpr (MODE == kForwardKeep) {
            u4 p[3];
            u4* to = planes + (i * S::FH + j) * 6 * 64;
            to_parts(x, p);
#pragma unroll
            for (int k = 0; k < 3; ++k) __builtin_nontemporal_store(p[k], to + k * 64);
            to_parts(y, p);
#pragma unroll
            for (int k = 0; k < 3; ++k) __builtin_nontemporal_store(p[k], to + (3 + k) * 64);
          }
          if constexpr (LOW) in_32_bits(h);
          to_rows(h, static_cast<T*>(a.out), a.F, m, n);
          if constexpr (LOW) to_rows(rest<T>(h), static_cast<T*>(a.out) + (int64_t)a.R * a.F, a.F, m, n);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    stored = inside;
  }
}

template <typename T, int MODE, int ACT, int BM, bool END, bool LOW = false> int launch_product_as(const GatedProductArgs& a, hipStream_t stream) {
  typedef GatedShape<MODE, BM> S;
  static PerDeviceOnce once;
  bool& configured = once.flag();
  if (!configured) {
    if (hipFuncSetAttribute(reinterpret_cast<const void*>(&gated_product_kernel<T, MODE, ACT, BM, END, LOW>), hipFuncAttributeMaxDynamicSharedMemorySize, S::kLds) != hipSuccess) return -3;
    configured = true;
  }
  const int64_t tiles = (int64_t)((a.R + BM - 1) / BM) * ((a.F + kTileF - 1) / kTileF);
  hipLaunchKernelGGL((gated_product_kernel<T, MODE, ACT, BM, END, LOW>), dim3((unsigned)std::min<int64_t>((tiles + 7) / 8 * 8, 256)), dim3(kWideThreads), S::kLds, stream, a);
  return hipGetLastError() == hipSuccess ? 0 : -3;
}
// Few numbers, 16-bit types: where h and [dg dv] alone are rounded on the way, results are 1.4 times as far from the formula as results rounded once, and of a few hundred numbers now and then twice as
// far.  There what the roundings leave takes part in the products too, and launches bound them as before (backward pass, us, rounded / in parts: 8 rows of 24 through 192 13.2 / 10.5, 5770 of 16 through 24
// 19.4 / 15.1, 40 of 96 through 4000 20.7 / 18.5; 1 of 1904 through 5048 51 / 61, whose gradients of 2 x 38 MB are written in pieces of 16 bytes.  Of that the look for what is not finite is 0.1 to 0.7).
bool few_numbers(int R, int D, int F) { return std::min({(int64_t)R * D, (int64_t)D * F, (int64_t)R * F}) < 4096; }
// Rows of a tile: those with which the fullest CU is done first (us a step of the contraction, and at a tile's end); of both passes, which share the order of a and b.
int tile_rows(int R, int D, int F) {
  if (few_numbers(R, D, F)) return 64;
  const int steps = (D + kWideK - 1) / kWideK;
  auto cost = [&](int rows, double step, double end) {
    const int64_t tiles = (int64_t)((R + rows - 1) / rows) * ((F + kTileF - 1) / kTileF);
    return (double)((tiles + 255) / 256) * (steps * step + end);
  };
  const double large = cost(256, 1.4, 5), middle = cost(128, 0.85, 3), small = cost(64, 0.56, 1.6);
  return small < std::min(middle, large) ? 64 : middle < large ? 128 : 256;
}
template <int MODE> int launch_product(const GatedProductArgs& a, int rows, int act, bool low, int dtype, hipStream_t stream) {
  return by_type16(dtype, true, [&](auto t, auto) {
    using T = decltype(t);
    if (low) {
      if constexpr (MODE != kBackward)
        if (act == kGeluGate) return launch_product_as<T, MODE, kGeluGate, 64, true, true>(a, stream);
      return launch_product_as<T, MODE, kSilu, 64, true, true>(a, stream);
    }
    auto of_end = [&](auto bm, auto ac) {
      constexpr int BM = decltype(bm)::value, ACT = decltype(ac)::value;
      return a.K % kWideK != 0 ? launch_product_as<T, MODE, ACT, BM, true>(a, stream) : launch_product_as<T, MODE, ACT, BM, false>(a, stream);
    };
    auto of_act = [&](auto bm) {
      if constexpr (MODE != kBackward)
        if (act == kGeluGate) return of_end(bm, std::integral_constant<int, kGeluGate>());
      return of_end(bm, std::integral_constant<int, kSilu>());   // (the backward pass has a and b)
    };
    return rows == 64 ? of_act(std::integral_constant<int, 64>()) : rows == 128 ? of_act(std::integral_constant<int, 128>()) : of_act(std::integral_constant<int, 256>());
  });
}

// ---- 16-bit types, few rows (tokens) ---------------------------------------------------------------------------------
// What bounds them is reading the weights once, and how many bytes the busiest CU draws (about 50 a ns): its rows of x and of the weights.  So every workgroup takes all rows and as many columns as let
// all CUs have one, both halves of them side by side, and its eight waves split the contraction, straight from memory to the matrix instructions, a few steps in flight at a time.  The second product,
// whose contraction is the long one, goes in ranges of it too, joined by a launch of its own.
// 32 rows of 2048 through 5504: 28.3 us with the tiles above and products in ranges, of which 19 and 11.5 on the GPU; here 24.9, of which 13.8 the first and 8.5 + 3.8 the second with its join.
constexpr int kFewRows = 64, kRowWaves = 8, kRowDepth = 32;   // rows at most, waves, contraction of a step
struct RowsArgs {
  const void *x, *w;
  int64_t ld_x, ld_w;
  int R, N, K, cols;     // cols: of a workgroup
  int64_t half;          // gate: elements from a row of w to the row of its other half
  int k_per_range;       // a multiple of kRowDepth
  void* out;             // [R][N]
  float* part;           // or partial results [range][out_R][N]
  int out_R;             // R; half of it: the rows of x are what has been rounded and, behind it, what that has left, and their sums are added
  bool low;              // gate: what the rounding of `out` leaves goes behind it
};
typedef vec<float, 4> acc4_t;
__device__ __forceinline__ void mma16(acc4_t& c, const vec<bf16_t, 8>& a, const vec<bf16_t, 8>& b) { c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ void mma16(acc4_t& c, const vec<fp16_t, 8>& a, const vec<fp16_t, 8>& b) { c = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
constexpr int kNoGate = -1;
// ACT: kNoGate, or tiles of 16 columns are 8 of either half.  MT: 16 rows each, NT: tiles of 16 columns
template <typename T, int ACT, int MT, int NT> __global__ __launch_bounds__(64 * kRowWaves, 2) void gated_rows_kernel(RowsArgs a) {
  extern __shared__ float s_sums[];   // [wave][16 MT][16 NT + 1]
  constexpr int LD = 16 * NT + 1, PER = ACT == kNoGate ? 16 : 8;   // columns of a tile
  constexpr int kRowSteps = MT + NT <= 5 ? 8 : 4;                  // in flight at a time: 160 registers
  typedef vec<T, 8> vt;
  const int lane = lane_id(), wave = wave_id(), c = lane & 15, g = lane >> 4, n0 = blockIdx.x * a.cols, n_end = min(a.N, n0 + a.cols);
  const int k0 = blockIdx.y * a.k_per_range, k1 = min(a.K, k0 + a.k_per_range), steps = (k1 - k0 + kRowDepth - 1) / kRowDepth, per = (steps + kRowWaves - 1) / kRowWaves;
  const int s_end = min(steps, (wave + 1) * per);
  const T *x = static_cast<const T*>(a.x) + k0 + 8 * g, *w = static_cast<const T*>(a.w) + k0 + 8 * g;
  const T* wr[NT];
  bool there[NT];
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    const int n = n0 + PER * j + (c & (PER - 1));
    there[j] = n < n_end;
    wr[j] = w + (int64_t)min(n, a.N - 1) * a.ld_w + (ACT != kNoGate && c >= 8 ? a.half : 0);
  }
  acc4_t acc[MT][NT];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j) acc[i][j] = acc4_t{0.f, 0.f, 0.f, 0.f};
  for (int s0 = wave * per; s0 < s_end; s0 += kRowSteps) {
    vt fa[kRowSteps][MT], fb[kRowSteps][NT];
#pragma unroll
    for (int u = 0; u < kRowSteps; ++u) {
      const int k = kRowDepth * (s0 + u);
      const bool in = s0 + u < s_end && k0 + k + 8 * g < k1;   // (whole pieces: K is a multiple of 8)
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        fb[u][j] = vt{};
        if (in && there[j]) fb[u][j] = *reinterpret_cast<const vt*>(wr[j] + k);
      }
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        fa[u][i] = vt{};
        if (in && 16 * i + c < a.R) fa[u][i] = *reinterpret_cast<const vt*>(x + (16 * i + c) * a.ld_x + k);
      }
    }
#pragma unroll
    for (int u = 0; u < kRowSteps; ++u)
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) mma16(acc[i][j], fa[u][i], fb[u][j]);
  }
  settle();
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int r = 0; r < 4; ++r) s_sums[(wave * 16 * MT + 16 * i + 4 * g + r) * LD + 16 * j + c] = acc[i][j][r];
  __syncthreads();
  auto sum = [&](int row, int col) __attribute__((always_inline)) {
    float v = 0.f;
#pragma unroll
    for (int k = 0; k < kRowWaves; ++k) v += s_sums[(k * 16 * MT + row) * LD + col];
    return v;
  };
  for (int o = threadIdx.x; o < 16 * MT * PER * NT; o += 64 * kRowWaves) {
    const int row = o / (PER * NT), col = o % (PER * NT), n = n0 + col;
    if (row >= a.out_R || n >= n_end) continue;
    if constexpr (ACT != kNoGate) {
      const int at = col / 8 * 16 + col % 8;
      float h = Gate<T, ACT>(sum(row, at)).act * sum(row, at + 8);
      in_32_bits(h);
      static_cast<T*>(a.out)[(int64_t)row * a.N + n] = (T)h;
      if (a.low) static_cast<T*>(a.out)[(int64_t)(a.R + row) * a.N + n] = (T)rest<T>(h);
    } else {
      float v = sum(row, col);
      if (a.out_R < a.R && __builtin_isfinite(v)) v += sum(a.out_R + row, col);   // (else the rest, zeros, may have met an infinity of the weights)
      if (a.part != nullptr) a.part[((int64_t)blockIdx.y * a.out_R + row) * a.N + n] = v;
      else static_cast<T*>(a.out)[(int64_t)row * a.N + n] = (T)v;
    }
  }
}
// Columns of a workgroup and ranges of the contraction: the least of what the busiest CU draws, and a launch to join ranges
struct RowsPlan { int cols, ranges; };
RowsPlan rows_plan(int R, int N, int K, bool gate) {
  const int halves = gate ? 2 : 1, most = 48 / halves;   // (three tiles of 16)
  RowsPlan best = {most, 1};
  double best_cost = 1e30;
  for (int ranges = 1; ranges <= (gate ? 1 : 8); ++ranges) {
    if (ranges > 1 && K / ranges < 2 * kRowDepth * kRowWaves) break;
    for (int cols = 4; cols <= most; ++cols) {
      const int64_t groups = (int64_t)((N + cols - 1) / cols) * ranges, turns = (groups + 255) / 256;
      const double cost = turns * (R + halves * cols) * (2.0 * K / ranges) / 50e3 + (ranges > 1 ? 3.0 + ranges * 8.0 * R * N / 4e6 : 0);
      if (cost < best_cost) {
        best_cost = cost;
        best = {cols, ranges};
      }
    }
  }
  return best;
}
template <typename T, int ACT> int launch_rows_as(const RowsArgs& a, int ranges, hipStream_t stream) {
  const int nt = (a.cols * (ACT == kNoGate ? 1 : 2) + 15) / 16;
  auto go = [&](auto m, auto n) {
    constexpr int MT = decltype(m)::value, NT = decltype(n)::value, kLds = kRowWaves * 16 * MT * (16 * NT + 1) * 4;
    static PerDeviceOnce once;
    bool& configured = once.flag();
    if (!configured) {
      if (hipFuncSetAttribute(reinterpret_cast<const void*>(&gated_rows_kernel<T, ACT, MT, NT>), hipFuncAttributeMaxDynamicSharedMemorySize, kLds) != hipSuccess) return -3;
      configured = true;
    }
    hipLaunchKernelGGL((gated_rows_kernel<T, ACT, MT, NT>), dim3((a.N + a.cols - 1) / a.cols, ranges), dim3(64 * kRowWaves), kLds, stream, a);
    return hipGetLastError() == hipSuccess ? 0 : -3;
  };
  auto of_rows = [&](auto m) {
    return nt == 1 ? go(m, std::integral_constant<int, 1>()) : nt == 2 ? go(m, std::integral_constant<int, 2>()) : go(m, std::integral_constant<int, 3>());
  };
  return a.R <= 16 ? of_rows(std::integral_constant<int, 1>()) : a.R <= 32 ? of_rows(std::integral_constant<int, 2>()) : of_rows(std::integral_constant<int, 4>());
}
// low: h, rounded, and behind it what that has left, is written (gate) or read
int64_t rows_bytes(int R, int N, int K, bool low) {
  const RowsPlan p = rows_plan(low ? 2 * R : R, N, K, false);
  return p.ranges > 1 ? ((int64_t)p.ranges * R * N * 4 + 255) / 256 * 256 : 0;
}
// act: kNoGate, or that of the gate between the two halves of w, N rows each
int launch_rows(const void* x, int64_t ld_x, const void* w, int64_t ld_w, void* out, int R, int N, int K, int act, bool low, int dtype, void* workspace, hipStream_t stream) {
  const int rows = low && act == kNoGate ? 2 * R : R;
  const RowsPlan p = rows_plan(rows, N, K, act != kNoGate);
  const int per = ((K + p.ranges - 1) / p.ranges + kRowDepth - 1) / kRowDepth * kRowDepth, ranges = (K + per - 1) / per;
  const RowsArgs a = {x, w, ld_x, ld_w, rows, N, K, p.cols, (int64_t)N * ld_w, per, out, ranges > 1 ? static_cast<float*>(workspace) : nullptr, R, low};
  const int rc = by_type16(dtype, true, [&](auto t, auto) {
    using T = decltype(t);
    return act == kNoGate ? launch_rows_as<T, kNoGate>(a, ranges, stream) : act == kSilu ? launch_rows_as<T, kSilu>(a, 1, stream) : launch_rows_as<T, kGeluGate>(a, 1, stream);
  });
  return rc != 0 || ranges == 1 ? rc : launch_part_sum(a.part, ranges, (int64_t)R * N, out, dtype, stream);
}

// ---- 16-bit types, few numbers ---------------------------------------------------------------------------------------
// Products of an operand in two parts, rounded and what that has left, with one in one: tiles of 32 x 32, four waves that take steps of 16 of the contraction in turns, straight from memory (16 bytes
// where the contraction is contiguous, else element by element, whose lanes lie side by side), in ranges that fill the card, summed in a launch of their own.
// What has left nothing is a zero, and makes a NaN of an infinity of the other operand.  So where sums are not finite, those of the rounded part alone count, formed again.
struct PartsJob {
  const void *a, *low, *b;   // a and low [M][lda] or [K][lda], b [N][ldb] or [K][ldb]
  int64_t lda, ldb, cm, cn;  // element (m, n) of c at m cm + n cn; one of them is 1
  int M, N, K, ranges, k_per_range;   // k_per_range: a multiple of 16
  void* c;
  float* part;               // [range], in c's order
};
struct PartsArgs {
  PartsJob job[3];
  int groups[3];
};
// eight steps of the contraction of one row or column.  LAST: those behind its end are zeros (none of what memory holds there meets anything).  All are requested, then looked at.
template <typename T, bool KC> struct PartsPiece {
  vec<uint32_t, KC ? 4 : 8> w;
  template <bool LAST> __device__ __forceinline__ void load(const T* p, int64_t ld, int k, int k_end) {
    if constexpr (KC) {
      w = *reinterpret_cast<const vec<uint32_t, 4>*>(p + (LAST ? min(k, k_end - 8) : k));   // (the contraction is a multiple of 8)
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) w[e] = reinterpret_cast<const uint16_t*>(p)[(int64_t)(LAST ? min(k + e, k_end - 1) : k + e) * ld];
    }
  }
  template <bool LAST> __device__ __forceinline__ frag<T> get(int k, int k_end) {
    if constexpr (LAST) {
#pragma unroll
      for (int e = 0; e < (KC ? 4 : 8); ++e) {
        uint32_t v = w[e];
        asm("" : "+v"(v));   // (a request by itself, not one behind a condition)
        w[e] = (KC ? k : k + e) < k_end ? v : 0u;
      }
    }
    if constexpr (KC) return __builtin_bit_cast(frag<T>, w);
    vec<uint32_t, 4> pairs;
#pragma unroll
    for (int e = 0; e < 4; ++e) pairs[e] = w[(KC ? 0 : 2) * e] | w[(KC ? 0 : 2) * e + (KC ? 0 : 1)] << 16;
    return __builtin_bit_cast(frag<T>, pairs);
  }
};
constexpr int kPartsWaves = 4;
// the waves of a workgroup share a tile, or, for short contractions, each has one
__host__ __device__ __forceinline__ bool parts_shared(int K) { return K > 64; }
template <typename T, bool AKC, bool BKC> __device__ __forceinline__ void parts_tile(const PartsJob& j, int group, vec<float, 4>* s_sum) {
  constexpr int U = 4;   // steps in flight
  const int lane = lane_id(), wave = wave_id(), c = lane & 31, g = lane >> 5;
  const bool shared = parts_shared(j.K);
  const int tiles_n = (j.N + 31) / 32, tiles = (j.M + 31) / 32 * tiles_n, range = shared ? group / tiles : 0, tile = shared ? group % tiles : group * kPartsWaves + wave;
  if (tile >= tiles) return;   // (not of a tile that waves share)
  const int m0 = tile / tiles_n * 32, n0 = tile % tiles_n * 32, m = min(m0 + c, j.M - 1), n = min(n0 + c, j.N - 1);   // (rows and columns behind the end: the last one's, not stored)
  const int k_end = min(j.K, (range + 1) * j.k_per_range), step = shared ? 16 * kPartsWaves : 16;
  const T *a = static_cast<const T*>(j.a) + (AKC ? m * j.lda : m), *low = static_cast<const T*>(j.low) + (AKC ? m * j.lda : m), *b = static_cast<const T*>(j.b) + (BKC ? n * j.ldb : n);
  acc_t acc;   // [n rows, m lanes]
  int k;
  auto steps = [&](auto u_, auto last_, auto both_) __attribute__((always_inline)) {
    constexpr int N = decltype(u_)::value;
    constexpr bool LAST = decltype(last_)::value, BOTH = decltype(both_)::value;
    PartsPiece<T, AKC> pa[N], pl[N];
    PartsPiece<T, BKC> pb[N];
#pragma unroll
    for (int u = 0; u < N; ++u) {
      const int at = k + step * u + 8 * g;
      pa[u].template load<LAST>(a, j.lda, at, k_end);
      if constexpr (BOTH) pl[u].template load<LAST>(low, j.lda, at, k_end);
      pb[u].template load<LAST>(b, j.ldb, at, k_end);
    }
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int u = 0; u < N; ++u) {
      const int at = k + step * u + 8 * g;
      const frag<T> fb = pb[u].template get<LAST>(at, k_end);
      if constexpr (BOTH) mma(acc, fb, pl[u].template get<LAST>(at, k_end));
      mma(acc, fb, pa[u].template get<LAST>(at, k_end));
    }
    k += step * N;
  };
  auto sums = [&](auto both) __attribute__((always_inline)) {
    zero(acc);
    k = range * j.k_per_range + (shared ? 16 * wave : 0);
    while (k + step * (U - 1) + 16 <= k_end) steps(std::integral_constant<int, U>(), std::false_type(), both);
    while (k < k_end) steps(std::integral_constant<int, 2>(), std::true_type(), both);
    settle();
  };
  sums(std::true_type());
  float most = 0.f;   // NaN where something is not finite
#pragma unroll
  for (int r = 0; r < 16; ++r) most += 0.f * acc[r];
  if (__ballot(most != 0.f) != 0) {
    const acc_t both = acc;
    sums(std::false_type());
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[r] = __builtin_isfinite((float)both[r]) ? both[r] : acc[r];
  }
  auto store = [&](const vec<float, 4>& x, int q) __attribute__((always_inline)) {
    const int64_t row = m0 + c, col = n0 + 8 * q + 4 * g, at = row * j.cm + col * j.cn;
    if (row >= j.M || col >= j.N) return;   // (columns are multiples of 8)
    auto to = [&](auto* out) __attribute__((always_inline)) {
      using O = std::remove_reference_t<decltype(*out)>;
      if (j.cn == 1) {
        *reinterpret_cast<vec<O, 4>*>(out + at) = __builtin_convertvector(x, vec<O, 4>);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) out[at + e * j.cn] = (O)(float)x[e];
      }
    };
    if (j.part != nullptr) to(j.part + (int64_t)range * j.M * j.N);
    else to(static_cast<T*>(j.c));
  };
  if (!shared) {
#pragma unroll
    for (int q = 0; q < 4; ++q) store(pack4<float>(acc, q), q);
    return;
  }
#pragma unroll
  for (int q = 0; q < 4; ++q) s_sum[(wave * 4 + q) * 64 + lane] = pack4<float>(acc, q);
  __syncthreads();
  vec<float, 4> x = s_sum[wave * 64 + lane];   // quad `wave` of all waves
#pragma unroll
  for (int w = 1; w < kPartsWaves; ++w) x += s_sum[(w * 4 + wave) * 64 + lane];
  store(x, wave);
}
template <typename T> __global__ __launch_bounds__(64 * kPartsWaves) void parts_product_kernel(PartsArgs p) {
  __shared__ vec<float, 4> s_sum[kPartsWaves * 4 * 64];
  parts_tile<T, true, true>(p.job[0], blockIdx.x, s_sum);
}
// the first job: dx, the others: weight gradients
template <typename T> __global__ __launch_bounds__(64 * kPartsWaves) void parts_grads_kernel(PartsArgs p) {
  __shared__ vec<float, 4> s_sum[kPartsWaves * 4 * 64];
  int group = blockIdx.x;
  if (group < p.groups[0]) {
    parts_tile<T, true, false>(p.job[0], group, s_sum);
  } else {
    group -= p.groups[0];
    const bool last = group >= p.groups[1];
    parts_tile<T, false, false>(p.job[last ? 2 : 1], last ? group - p.groups[1] : group, s_sum);
  }
}
// ranges of a job, its workgroups; what its partial sums take
int64_t parts_plan(PartsJob& j, int& groups) {
  const int64_t tiles = (int64_t)((j.M + 31) / 32) * ((j.N + 31) / 32);
  const int steps = (j.K + 15) / 16, most = (int)std::max<int64_t>(1, std::min<int64_t>({512 / tiles, 128, steps / (4 * kPartsWaves)}));
  if (!parts_shared(j.K)) {
    j.k_per_range = 64;
    j.ranges = 1;
    groups = (int)((tiles + kPartsWaves - 1) / kPartsWaves);
    return 0;
  }
  const int each = (steps + most - 1) / most;
  j.k_per_range = 16 * each;
  j.ranges = (steps + each - 1) / each;
  groups = (int)(tiles * j.ranges);
  return j.ranges > 1 ? ((int64_t)j.ranges * j.M * j.N * 4 + 255) / 256 * 256 : 0;
}
int64_t parts_bytes(int M, int N, int K) {
  PartsJob j = {};
  j.M = M;
  j.N = N;
  j.K = K;
  int groups;
  return parts_plan(j, groups);
}
template <typename Launch> int launch_parts(PartsArgs& p, int dtype, void* workspace, hipStream_t stream, Launch&& launch) {
  char* at = static_cast<char*>(workspace);
  PartSum sums[3];
  int count = 0, groups = 0;
  for (int i = 0; i < 3; ++i) {
    PartsJob& j = p.job[i];
    p.groups[i] = 0;
    if (j.c == nullptr) continue;
    const int64_t bytes = parts_plan(j, p.groups[i]);
    groups += p.groups[i];
    if (bytes == 0) continue;
    j.part = reinterpret_cast<float*>(at);
    at += bytes;
    sums[count++] = {j.part, (int64_t)j.M * j.N, j.c, j.ranges, 0};
  }
  const int rc = by_type16(dtype, true, [&](auto t, auto) {
    launch(t, groups);
    return hipGetLastError() == hipSuccess ? 0 : -3;
  });
  return rc != 0 || count == 0 ? rc : launch_sums(sums, count, dtype, stream);
}

int64_t up(int64_t n) { return (n + 255) / 256 * 256; }
int elem_size(int dtype) { return dtype == 0 ? 4 : 2; }

struct Operand2 {
  const void* p;
  int64_t ld;
  bool kc;   // contraction-contiguous
};
int64_t product_workspace(int M, int N, int K, int dtype) { return up(gemm_workspace(M, N, K, elem_size(dtype), false)); }
GemmArgs product_args(const Operand2& a, const Operand2& b, void* c, int M, int N, int K) {
  return {a.p, b.p, c, nullptr, M, N, K, a.ld, b.ld, N, kGemmPlain, 0, nullptr, nullptr, nullptr, 0, 1, nullptr, 0.f, nullptr, nullptr};
}
int product(const Operand2& a, const Operand2& b, void* c, int M, int N, int K, int dtype, void* workspace, hipStream_t stream) {
  const GemmArgs g = product_args(a, b, c, M, N, K);
  return launch_gemm(g, a.kc, b.kc, dtype, static_cast<float*>(workspace), stream);
}
// Gradients of a projection y = x w^T, dy [R][N], x [R][K], and `more`, the weight gradient of another one of as many rows: of what is asked for (c not nullptr) as much in one launch as is ahead so
struct More {
  Operand2 a, b;
  void* c;
  int M, N;
};
int64_t grads_bytes(int R, int N, int K, int dtype, bool dw, bool dx, int more_m, int more_n) {
  const int64_t more = more_m > 0 ? product_workspace(more_m, more_n, R, dtype) : 0, both = dw && dx ? grads_workspace(R, N, K, elem_size(dtype), kGemmPlain, false) : -1;
  if (both < 0) return std::max({dw ? product_workspace(N, K, R, dtype) : 0, dx ? product_workspace(R, K, N, dtype) : 0, more});
  const int64_t third = more_m > 0 ? grads_more(R, N, K, elem_size(dtype), more_m, more_n) : -1;
  return third >= 0 ? up(both + third) : std::max(up(both), more);
}
int grads(const Operand2& dy, const Operand2& x, const Operand2& w, void* dw, void* dx, int R, int N, int K, const More& more, int dtype, void* workspace, hipStream_t stream) {
  if (dw != nullptr && dx != nullptr && grads_workspace(R, N, K, elem_size(dtype), kGemmPlain, false) >= 0) {
    MoreGradsArgs p = {};
    p.w = product_args(dy, x, dw, N, K, R);
    p.x = product_args(dy, w, dx, R, K, N);
    if (more.c == nullptr) return launch_grads(p, dtype, static_cast<float*>(workspace), nullptr, stream);
    if (grads_more(R, N, K, elem_size(dtype), more.M, more.N) >= 0) {
      p.v = product_args(more.a, more.b, more.c, more.M, more.N, R);
      return launch_more_grads(p, dtype, static_cast<float*>(workspace), stream);
    }
    const int rc = product(more.a, more.b, more.c, more.M, more.N, R, dtype, workspace, stream);
    return rc != 0 ? rc : launch_grads(p, dtype, static_cast<float*>(workspace), nullptr, stream);
  }
  int rc = 0;
  if (more.c != nullptr) rc = product(more.a, more.b, more.c, more.M, more.N, R, dtype, workspace, stream);
  if (rc == 0 && dx != nullptr) rc = product({dy.p, dy.ld, true}, {w.p, w.ld, false}, dx, R, K, N, dtype, workspace, stream);
  if (rc == 0 && dw != nullptr) rc = product({dy.p, dy.ld, false}, {x.p, x.ld, false}, dw, N, K, R, dtype, workspace, stream);
  return rc;
}

// f(activation)
template <typename F> int by_act(int act, F&& f) { return act == kSilu ? f(std::integral_constant<int, kSilu>()) : f(std::integral_constant<int, kGeluGate>()); }

// Both weight gradients in one launch, where that is ahead of one for each (the second of which may be that of dx too); all: dx is in it too
bool both_weights(int R, int D, int F, int dtype, bool dx, WeightsPlan& p, bool& all) {
  all = false;
  if (dtype == 0 || (dx && grads_workspace(R, 2 * F, D, 2, kGemmPlain, false) >= 0)) return false;
  p = weights_plan(R, 2 * F, D, D, F);
  const float weights = gemm_cost(2 * F, D, R, 2) + gemm_cost(D, F, R, 2);
  if (dx) {
    const WeightsPlan q = gradients_plan(R, 2 * F, D, D, F, R, D, 2 * F);
    all = q.cost < 0.9f * (std::min(p.cost, weights) + gemm_cost(R, D, 2 * F, 2));
    if (all) p = q;
  }
  return all || p.cost < weights;
}

bool few_rows(int R, int dtype) { return R <= kFewRows && dtype != 0; }
bool in_parts(int R, int D, int F, int dtype) { return dtype != 0 && few_numbers(R, D, F); }
// of h; and, in parts, of what its rounding has left
int64_t hidden_bytes(int R, int D, int F, int dtype) { return up((int64_t)R * F * elem_size(dtype) * (in_parts(R, D, F, dtype) ? 2 : 1)); }
int64_t planes_bytes(int R, int D, int F) {
  const int rows = tile_rows(R, D, F);
  return (int64_t)((R + rows - 1) / rows) * ((F + kTileF - 1) / kTileF) * rows * kTileF * 6;
}

}  // namespace

// What the backward pass needs: fp32 u, [R][2 F]; else h, [R][F], and a and b
int64_t gated_state(int R, int D, int F, int dtype) { return dtype == 0 ? 2 * hidden_bytes(R, D, F, 0) : hidden_bytes(R, D, F, dtype) + planes_bytes(R, D, F); }
// y is a product of all rows in a workgroup
bool down_by_rows(int R, int D, int F, int dtype) { return few_rows(in_parts(R, D, F, dtype) ? 2 * R : R, dtype); }
int64_t gated_workspace(int R, int D, int F, int dtype, bool keeps) {
  const bool parts = in_parts(R, D, F, dtype);
  const int64_t h = hidden_bytes(R, D, F, dtype), down = down_by_rows(R, D, F, dtype) ? rows_bytes(R, D, F, parts) : parts ? parts_bytes(R, D, F) : product_workspace(R, D, F, dtype);
  if (dtype != 0) return std::max<int64_t>(256, (keeps ? 0 : h) + down);
  if (gate_on_store(R, 2 * F, D)) return h + down;
  return h + (keeps ? 0 : 2 * h) + std::max(product_workspace(R, 2 * F, D, 0), down);
}
int launch_gated(const GatedArgs& a, void* y, void* state, int dtype, void* workspace, hipStream_t stream) {
  char* at = static_cast<char*>(workspace);
  const int64_t hidden = hidden_bytes(a.R, a.D, a.F, dtype);
  const bool parts = in_parts(a.R, a.D, a.F, dtype), by_rows = down_by_rows(a.R, a.D, a.F, dtype);
  auto take = [&](int64_t bytes) { char* p = at; at += bytes; return p; };
  void* h;
  int rc;
  if (dtype != 0) {
    h = state != nullptr ? state : take(hidden);
    const GatedProductArgs p = {a.x, a.w_in, a.ld_x, a.ld_in, a.R, a.F, a.D, h, state != nullptr ? static_cast<unsigned char*>(state) + hidden : nullptr};
    const int rows = tile_rows(a.R, a.D, a.F);
    if (state != nullptr) rc = launch_product<kForwardKeep>(p, rows, a.act, parts, dtype, stream);
    else if (by_rows) rc = launch_rows(a.x, a.ld_x, a.w_in, a.ld_in, h, a.R, a.F, a.D, a.act, parts, dtype, nullptr, stream);
    else rc = launch_product<kForward>(p, rows, a.act, parts, dtype, stream);
  } else {
    h = take(hidden);
    const int64_t n = (int64_t)a.R * a.F;
    const bool fused = gate_on_store(a.R, 2 * a.F, a.D);
    float* u = static_cast<float*>(state != nullptr ? state : fused ? nullptr : take(2 * hidden));
    if (fused) {
      GemmArgs g = product_args({a.x, a.ld_x, true}, {a.w_in, a.ld_in, true}, u, a.R, 2 * a.F, a.D);
      g.h = h;
      rc = launch_gemm_gate(g, kGateForward, a.act, stream);
    } else {
      rc = product({a.x, a.ld_x, true}, {a.w_in, a.ld_in, true}, u, a.R, 2 * a.F, a.D, dtype, at, stream);
      if (rc == 0)
        rc = by_act(a.act, [&](auto act) {
          hipLaunchKernelGGL((gate_kernel<decltype(act)::value>), many_blocks((n / 8 + kThreads - 1) / kThreads), dim3(kThreads), 0, stream, u, n, a.F, static_cast<float*>(h));
          return hipGetLastError() == hipSuccess ? 0 : -3;
        });
    }
  }
  if (rc != 0) return rc;
  if (by_rows) return launch_rows(h, a.F, a.w_out, a.ld_out, y, a.R, a.D, a.F, kNoGate, parts, dtype, at, stream);
  if (parts) {
    PartsArgs p = {};
    p.job[0] = {h, static_cast<const uint16_t*>(h) + (int64_t)a.R * a.F, a.w_out, a.F, a.ld_out, a.D, 1, a.R, a.D, a.F, 0, 0, y, nullptr};
    return launch_parts(p, dtype, at, stream, [&](auto t, int groups) { hipLaunchKernelGGL((parts_product_kernel<decltype(t)>), dim3(groups), dim3(64 * kPartsWaves), 0, stream, p); });
  }
  return product({h, a.F, true}, {a.w_out, a.ld_out, true}, y, a.R, a.D, a.F, dtype, at, stream);
}

int64_t gated_bwd_workspace(int R, int D, int F, int dtype, int gradients) {
  const bool dx = gradients & 1, dw_in = gradients & 2, dw_out = gradients & 4, below = dx || dw_in;
  const int64_t hidden = hidden_bytes(R, D, F, dtype);
  int64_t products = grads_bytes(R, 2 * F, D, dtype, dw_in, dx, dw_out ? D : 0, F);
  WeightsPlan p;
  bool all;
  if (dw_in && dw_out && both_weights(R, D, F, dtype, dx, p, all)) products = std::max(up(weights_workspace(p)), dx && !all ? product_workspace(R, D, 2 * F, dtype) : 0);
  if (in_parts(R, D, F, dtype)) products = (dx ? parts_bytes(R, D, 2 * F) : 0) + (dw_in ? parts_bytes(2 * F, D, R) : 0) + (dw_out ? parts_bytes(F, D, R) : 0);
  if (dtype != 0) return std::max<int64_t>(256, (below ? 2 * hidden : 0) + products);
  const int64_t h = dw_out ? hidden : 0;
  if (!below) return std::max<int64_t>(256, h + products);
  return gate_on_store(R, F, D) ? h + 2 * hidden + products : h + 3 * hidden + std::max(products, product_workspace(R, F, D, 0));
}
int launch_gated_bwd(const GatedArgs& a, const void* dy, const void* state, void* dx, void* dw_in, void* dw_out, int dtype, void* workspace, hipStream_t stream) {
  char* at = static_cast<char*>(workspace);
  const int64_t hidden = hidden_bytes(a.R, a.D, a.F, dtype), n = (int64_t)a.R * a.F;
  const bool below = dx != nullptr || dw_in != nullptr, parts = in_parts(a.R, a.D, a.F, dtype);
  auto take = [&](int64_t bytes) { char* p = at; at += bytes; return p; };
  const void* h = state;
  void* du = nullptr;
  int rc = 0;
  if (dtype != 0) {
    if (below) {
      du = take(2 * hidden);
      const GatedProductArgs p = {dy, a.w_out, a.D, a.ld_out, a.R, a.F, a.D, du, const_cast<unsigned char*>(static_cast<const unsigned char*>(state)) + hidden};
      rc = launch_product<kBackward>(p, tile_rows(a.R, a.D, a.F), a.act, parts, dtype, stream);
    }
  } else {
    float* h32 = dw_out != nullptr ? reinterpret_cast<float*>(take(hidden)) : nullptr;
    const float* dh = nullptr;
    h = h32;
    const bool fused = below && gate_on_store(a.R, a.F, a.D);
    if (fused) {
      du = take(2 * hidden);
      GemmArgs g = product_args({dy, a.D, true}, {a.w_out, a.ld_out, false}, du, a.R, a.F, a.D);
      g.aux = const_cast<void*>(state);
      g.ldc = 2 * a.F;
      g.h = h32;
      rc = launch_gemm_gate(g, kGateBackward, a.act, stream);
    } else if (below) {
      dh = reinterpret_cast<const float*>(take(hidden));
      du = take(2 * hidden);
      rc = product({dy, a.D, true}, {a.w_out, a.ld_out, false}, const_cast<float*>(dh), a.R, a.F, a.D, dtype, at, stream);
    }
    if (rc == 0 && !fused)
      rc = by_act(a.act, [&](auto act) {
        hipLaunchKernelGGL((gate_bwd_kernel<decltype(act)::value>), many_blocks((n / 8 + kThreads - 1) / kThreads), dim3(kThreads), 0, stream, static_cast<const float*>(state), dh, n, a.F,
                           static_cast<float*>(du), h32);
        return hipGetLastError() == hipSuccess ? 0 : -3;
      });
  }
  if (parts) {
    if (rc != 0) return rc;
    const uint16_t *d = static_cast<const uint16_t*>(du), *hh = static_cast<const uint16_t*>(h);
    const int64_t n2 = 2 * n;
    PartsArgs p = {};
    if (dx != nullptr) p.job[0] = {d, d + n2, a.w_in, 2 * (int64_t)a.F, a.ld_in, a.D, 1, a.R, a.D, 2 * a.F, 0, 0, dx, nullptr};
    if (dw_in != nullptr) p.job[1] = {d, d + n2, a.x, 2 * (int64_t)a.F, a.ld_x, a.D, 1, 2 * a.F, a.D, a.R, 0, 0, dw_in, nullptr};
    if (dw_out != nullptr) p.job[2] = {hh, hh + n, dy, a.F, a.D, 1, a.F, a.F, a.D, a.R, 0, 0, dw_out, nullptr};
    return launch_parts(p, dtype, at, stream, [&](auto t, int groups) { hipLaunchKernelGGL((parts_grads_kernel<decltype(t)>), dim3(groups), dim3(64 * kPartsWaves), 0, stream, p); });
  }
  WeightsPlan plan;
  bool all;
  if (rc == 0 && dw_in != nullptr && dw_out != nullptr && both_weights(a.R, a.D, a.F, dtype, dx != nullptr, plan, all)) {
    const WeightProduct x = {du, a.w_in, dx, a.R, a.D, 2 * a.F, a.ld_in};
    rc = launch_weights({du, a.x, dw_in, 2 * a.F, a.D, 2 * a.F, a.ld_x}, {dy, h, dw_out, a.D, a.F, a.D, a.F}, all ? &x : nullptr, 2 * a.F, a.R, plan, dtype, reinterpret_cast<float*>(at), stream);
    return rc != 0 || dx == nullptr || all ? rc : product({du, 2 * a.F, true}, {a.w_in, a.ld_in, false}, dx, a.R, a.D, 2 * a.F, dtype, at, stream);
  }
  if (rc != 0) return rc;
  return grads({du, 2 * a.F, true}, {a.x, a.ld_x, true}, {a.w_in, a.ld_in, true}, dw_in, dx, a.R, 2 * a.F, a.D, {{dy, a.D, false}, {h, a.F, false}, dw_out, a.D, a.F}, dtype, at, stream);
}

}  // namespace castle
