// Two weight gradients of the same rows in one launch, 16-bit types: c = a^T b for a [R][M] and b [R][N], twice.
// By itself each has few tiles for its contraction, or some hundred for 256 CUs, with a last round that leaves most of them idle.  Here the tiles of both are one list.  So many as fill whole rounds of
// the card are taken whole; the others are cut into equal ranges of the contraction such that these fill rounds as well, and a second kernel adds the ranges' sums in their order.  The ranges of one
// part of the contraction stand side by side in the list: the workgroups of an XCD read the same rows of all operands, which its L2 holds.
// The frame is that of gemm_wide_kernel (castle_gemm.hip).  What bounds it: a step of 64 rows of a 256 x 256 tile takes 1.56 us, 1.38 PFLOP/s on all CUs, at the power that the matrix
// instructions are given.  16384 rows of 512 through 1408, 34 tiles: two products in 10 ranges each 98.3 us and their sums 16.8, here 238 ranges 79.3 and 12.2 (a third of the 79.3 is the end, where all
// write their sums at once, 62 MB).  8192 rows of 2048 through 5504, 520 tiles: 585 and 34 (344 and 176 tiles leave two thirds of a last round idle), here two rounds and 8 tiles in ranges, 471 and 8.
#include "castle_dispatch.h"
#include "castle_weights.h"
#include "castle_wide.h"
#include <algorithm>

namespace castle {
namespace {

constexpr int kTile = 256, kCus = 256, kPart = kTile * kTile;   // kPart: numbers of a range's sums
constexpr int kStage = 2 * kTile * kWideK * 2, kTurn = 4096, kLds = 2 * kStage + 8 * kTurn, kLoads = kStage / 1024 / 8;
static_assert(kLds <= kMaxLds, "");
__device__ const uint32_t castle_weights_zeros[4] __attribute__((aligned(16))) = {0, 0, 0, 0};
extern __shared__ __attribute__((aligned(16))) unsigned char castle_weights_lds[];

__host__ __device__ inline int tiles_of(int M, int N) { return (M + kTile - 1) / kTile * ((N + kTile - 1) / kTile); }

struct WeightsArgs {
  WeightProduct p[2];
  int tiles0, R, whole, rest, ranges, steps;
  float* part;   // of range q of tile whole + t: [q][t], in the order of the registers
};
// rows of a band of 2048 columns, then those of the next
__device__ __forceinline__ const WeightProduct& place(const WeightsArgs& a, int t, int& m0, int& n0) {
  const bool second = t >= a.tiles0;
  const WeightProduct& p = a.p[second];
  if (second) t -= a.tiles0;
  constexpr int kBand = 2048 / kTile;
  const int tiles_m = (p.M + kTile - 1) / kTile, tiles_n = (p.N + kTile - 1) / kTile, band = t / (tiles_m * kBand), rest = t - band * tiles_m * kBand, width = min(kBand, tiles_n - band * kBand);
  m0 = rest / width * kTile;
  n0 = (band * kBand + rest % width) * kTile;
  return p;
}

// END: the contraction ends inside a step
template <typename T, bool END> __global__ __launch_bounds__(kWideThreads, 2) void weights_kernel(WeightsArgs a) {
  typedef WideOperand<T, false, kTile> Op;
  typedef vec<T, 8> vt;
  const int lane = lane_id(), wave = wave_id(), c = lane & 31, g = lane >> 5, wm = wave / 2 * 64, wn = wave % 2 * 128;
  const int all_steps = (a.R + kWideK - 1) / kWideK, stride = gridDim.x, last = a.whole + a.rest * a.ranges;
  int unit = blockIdx.x % 8 * (stride / 8) + blockIdx.x / 8;   // XCD x takes the x-th eighth of a round
  if (unit >= last) return;
  const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) unsigned char*)castle_weights_lds;
  auto steps_of = [&](int u, int& tile, int& from) __attribute__((always_inline)) {
    tile = u;
    from = 0;
    if (u < a.whole) return all_steps;
    const int q = (u - a.whole) / a.rest;
    tile = u - q * a.rest;
    from = q * a.steps;
    return min(a.steps, all_steps - from);
  };
  // the step that is requested next runs ahead of the one that is multiplied, into the next tile or range
  Op ra, rb;
  int64_t lda, ldb;
  int next_unit = unit, next_step, next_end, ahead = 0;   // ahead: steps requested and not waited for
  auto start = [&]() __attribute__((always_inline)) {
    int tile, m0, n0;
    const int n = steps_of(next_unit, tile, next_step);
    next_end = next_step + n;
    const WeightProduct& p = place(a, tile, m0, n0);
    lda = p.lda;
    ldb = p.ldb;
    ra.start(static_cast<const T*>(p.a), lda, m0, p.M, next_step * kWideK);
    rb.start(static_cast<const T*>(p.b), ldb, n0, p.N, next_step * kWideK);
  };
  auto request = [&](int buffer) __attribute__((always_inline)) {
    if (next_unit >= last) return;
    ++ahead;
    if (END && next_step == all_steps - 1) {
      const int left = a.R - next_step * kWideK;
      ra.load_end(left, reinterpret_cast<const T*>(castle_weights_zeros), lds0 + buffer);
      rb.load_end(left, reinterpret_cast<const T*>(castle_weights_zeros), lds0 + buffer + kStage / 2);
    } else {
      ra.load(lda, lds0 + buffer);
      rb.load(ldb, lds0 + buffer + kStage / 2);
    }
    if (++next_step == next_end) {
      next_unit += stride;
      if (next_unit < last) start();
    }
  };
  start();
  request(0);
  request(kStage);
  // The step behind the current one is in LDS, from every wave, and all have read the current one.  A step and the stores of a tile inside its output, 16 or 32, come behind it and are not waited for.
  int stores = 0;
  auto arrive = [&]() __attribute__((always_inline)) {
    auto wait = [&](auto n) __attribute__((always_inline)) {
      asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(decltype(n)::value) : "memory");
    };
    if (ahead > 1) {
      if (stores == 2) wait(std::integral_constant<int, kLoads + 32>());
      else if (stores == 1) wait(std::integral_constant<int, kLoads + 16>());
      else wait(std::integral_constant<int, kLoads>());
    } else {
      if (stores == 2) wait(std::integral_constant<int, 32>());
      else if (stores == 1) wait(std::integral_constant<int, 16>());
      else wait(std::integral_constant<int, 0>());
    }
    stores = 0;
    --ahead;
  };
  int buffer = 0;
  frag<T> fa[2][2], fb[2][4];
  auto read = [&](int slot, int s) __attribute__((always_inline)) {
    const T* l = reinterpret_cast<const T*>(castle_weights_lds + buffer);
    Op::read(l, fa[slot], wm, s, c, g);
    Op::read(l + kTile * kWideK, fb[slot], wn, s, c, g);
    __builtin_amdgcn_sched_barrier(0);   // these reads, then the products of the fragments before
  };
  arrive();
  read(0, 0);
  for (; unit < last; unit += stride) {
    int tile, from, m0, n0;
    const int steps = steps_of(unit, tile, from);
    const WeightProduct& p = place(a, tile, m0, n0);
    acc_t acc[2][4];   // [n rows, m lanes]
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) zero(acc[i][j]);
    auto multiply = [&](int slot) __attribute__((always_inline)) {
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) mma(acc[i][j], fb[slot][j], fa[slot][i]);
    };
    int done = 0;   // buffer of the step that ends
    for (int it = 0; it < steps; ++it) {
#pragma unroll
      for (int s = 0; s < kWideK / 16 - 1; ++s) {
        read(1 - s % 2, s + 1);
        multiply(s % 2);
      }
      arrive();
      done = buffer;
      buffer = kStage - buffer;
      if (it + 1 < steps) request(done);
      read(0, 0);   // (behind the last step of all: what is there, for nothing)
      multiply(1);
    }
    asm volatile("s_nop 15\n\ts_nop 3" ::: "memory");   // the loop may end right behind a product
    __builtin_amdgcn_sched_barrier(0);
    request(done);
    if (unit >= a.whole && a.ranges > 1) {
      vec<float, 4>* part = reinterpret_cast<vec<float, 4>*>(a.part + (int64_t)(unit - a.whole) * kPart) + wave * 2048 + lane;
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int q = 0; q < 4; ++q) part[((i * 4 + j) * 4 + q) * 64] = pack4<float>(acc[i][j], q);
      stores = 2;
      continue;
    }
    // to whole rows, 32 rows of 64 columns at a time, each wave in a place of its own; piece k of row r at k ^ (r / 2 % 8)
    T* out = reinterpret_cast<T*>(castle_weights_lds + 2 * kStage + wave * kTurn);
#pragma unroll
    for (int h = 0; h < 4; ++h) {
      const int i = h % 2, half = h / 2;
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int q = 0; q < 4; ++q) st4<T>(out + c * 64 + 8 * ((4 * j + q) ^ (c >> 1 & 7)) + 4 * g, pack4<T>(acc[i][2 * half + j], q));
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int row = 8 * r + (lane >> 3), m = m0 + wm + 32 * i + row, n = n0 + wn + 64 * half + 8 * (lane & 7);
        const vt x = *reinterpret_cast<const vt*>(out + row * 64 + 8 * ((lane & 7) ^ (row >> 1 & 7)));
        if (m < p.M && n < p.N) *reinterpret_cast<vt*>(static_cast<T*>(p.c) + (int64_t)m * p.N + n) = x;
      }
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    if (m0 + kTile <= p.M && n0 + kTile <= p.N) stores = 1;
  }
}

// four columns a thread, in the order of the registers that they come from
template <typename T> __global__ __launch_bounds__(256) void weights_join_kernel(WeightsArgs a) {
  const int t = blockIdx.x / (kPart / 1024), at = blockIdx.x % (kPart / 1024) * 256 + threadIdx.x;
  const vec<float, 4>* part = reinterpret_cast<const vec<float, 4>*>(a.part) + (int64_t)t * (kPart / 4) + at;
  const int64_t next = (int64_t)a.rest * (kPart / 4);
  vec<float, 4> sum = part[0];
#pragma unroll 4
  for (int q = 1; q < a.ranges; ++q) sum += part[q * next];
  int m0, n0;
  const WeightProduct& p = place(a, a.whole + t, m0, n0);
  const int lane = at & 63, q = at >> 6 & 3, j = at >> 8 & 3, i = at >> 10 & 1, wave = at >> 11;
  const int m = m0 + wave / 2 * 64 + 32 * i + (lane & 31), n = n0 + wave % 2 * 128 + 32 * j + 8 * q + 4 * (lane >> 5);
  if (m < p.M && n < p.N) *reinterpret_cast<vec<T, 4>*>(static_cast<T*>(p.c) + (int64_t)m * p.N + n) = __builtin_convertvector(sum, vec<T, 4>);
}

template <typename T, bool END> int launch_kernel(const WeightsArgs& a, hipStream_t stream) {
  static PerDeviceOnce once;
  bool& configured = once.flag();
  if (!configured) {
    if (hipFuncSetAttribute(reinterpret_cast<const void*>(&weights_kernel<T, END>), hipFuncAttributeMaxDynamicSharedMemorySize, kLds) != hipSuccess) return -3;
    configured = true;
  }
  const int units = a.whole + a.rest * a.ranges;
  hipLaunchKernelGGL((weights_kernel<T, END>), dim3(std::min((units + 7) / 8 * 8, kCus)), dim3(kWideThreads), kLds, stream, a);
  return hipGetLastError() == hipSuccess ? 0 : -3;
}

}  // namespace

// us: a start, and for each round of the card so much a step and at the end of a tile or range; the ranges' sums are written and read
WeightsPlan weights_plan(int R, int M0, int N0, int M1, int N1) {
  const int64_t n64 = (int64_t)tiles_of(M0, N0) + tiles_of(M1, N1);
  const int steps = (R + kWideK - 1) / kWideK;
  WeightsPlan best = {0, 0, 1, steps, 1e30f};
  if (n64 > 1 << 20) return best;
  const int n = (int)n64;
  for (int whole = n / kCus * kCus, k = 0; whole >= 0 && k < 2; whole -= kCus, ++k) {
    const int rest = n - whole;
    for (int s = 1; s <= std::min(32, std::max(1, steps / 4)); ++s) {
      const int each = (steps + s - 1) / s, ranges = (steps + each - 1) / each;
      if (ranges != s || (int64_t)rest * s > 1024) continue;
      const int rounds = (rest * s + kCus - 1) / kCus;
      const float cost = 4 + whole / kCus * (steps * 1.56f + 4) + rounds * (each * 1.56f + 4) + (s > 1 ? 4 + rest * s * 0.09f : 0);
      if (cost < best.cost) best = {whole, rest, s, each, cost};
    }
  }
  return best;
}
int64_t weights_workspace(const WeightsPlan& p) { return p.ranges > 1 ? (int64_t)p.rest * p.ranges * kPart * 4 : 0; }

int launch_weights(const WeightProduct& first, const WeightProduct& second, int R, const WeightsPlan& p, int dtype, float* workspace, hipStream_t stream) {
  const WeightsArgs a = {{first, second}, tiles_of(first.M, first.N), R, p.whole, p.rest, p.ranges, p.steps, workspace};
  return by_type16(dtype, true, [&](auto t, auto) {
    using T = decltype(t);
    const int rc = R % kWideK == 0 ? launch_kernel<T, false>(a, stream) : launch_kernel<T, true>(a, stream);
    if (rc == 0 && p.ranges > 1) hipLaunchKernelGGL((weights_join_kernel<T>), dim3(p.rest * (kPart / 1024)), dim3(256), 0, stream, a);
    return rc != 0 ? rc : hipGetLastError() == hipSuccess ? 0 : -3;
  });
}

}  // namespace castle
