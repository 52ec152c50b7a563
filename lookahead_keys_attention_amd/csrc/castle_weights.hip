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
  // with the input gradient: dx [R][N] = a b for a [R][lda] and b [K][ldb]
  WeightProduct x;
  int x_groups, x_steps, longs, long_steps;   // x_groups: workgroups of an XCD that have a tile of it; x_steps: its whole contraction, K
};
// rows of a band of 2048 columns, then those of the next
__device__ __forceinline__ void place_in(const WeightProduct& p, int t, int& m0, int& n0) {
  constexpr int kBand = 2048 / kTile;
  const int tiles_m = (p.M + kTile - 1) / kTile, tiles_n = (p.N + kTile - 1) / kTile, band = t / (tiles_m * kBand), rest = t - band * tiles_m * kBand, width = min(kBand, tiles_n - band * kBand);
  m0 = rest / width * kTile;
  n0 = (band * kBand + rest % width) * kTile;
}
__device__ __forceinline__ WeightProduct place(const WeightsArgs& a, int t, int& m0, int& n0) {
  const bool second = t >= a.tiles0;
  const WeightProduct &x = a.p[0], &y = a.p[1];
  const WeightProduct p = {second ? y.a : x.a, second ? y.b : x.b, second ? y.c : x.c, second ? y.M : x.M, second ? y.N : x.N, second ? y.lda : x.lda, second ? y.ldb : x.ldb};
  place_in(p, second ? t - a.tiles0 : t, m0, n0);
  return p;
}

// What a workgroup does next: steps of a tile's contraction; slot: where the sums of a range go, -1: to the output.
struct Unit {
  WeightProduct p;
  int m0, n0, from, steps, slot;
};
// Units 0, 1, ... of the workgroup, as long as at(i, unit) has one.  AKC: a is contraction-contiguous.  K: the whole contraction, END: it ends inside a step.
template <typename T, bool AKC, bool END, typename At> __device__ __forceinline__ void run_units(At&& at, int K, float* parts) {
  typedef WideOperand<T, AKC, kTile> OpA;
  typedef WideOperand<T, false, kTile> OpB;
  typedef vec<T, 8> vt;
  const int lane = lane_id(), wave = wave_id(), c = lane & 31, g = lane >> 5, wm = wave / 2 * 64, wn = wave % 2 * 128;
  const int all_steps = (K + kWideK - 1) / kWideK;
  const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) unsigned char*)castle_weights_lds;
  Unit unit, next;
  if (!at(0, unit)) return;
  next = unit;
  // the step that is requested next runs ahead of the one that is multiplied, into the next tile or range
  OpA ra;
  OpB rb;
  int next_i = 0, next_step = 0, ahead = 0;   // ahead: steps requested and not waited for
  bool left = true;
  auto start = [&]() __attribute__((always_inline)) {
    next_step = next.from;
    ra.start(static_cast<const T*>(next.p.a), next.p.lda, next.m0, next.p.M, next_step * kWideK);
    rb.start(static_cast<const T*>(next.p.b), next.p.ldb, next.n0, next.p.N, next_step * kWideK);
  };
  auto request = [&](int buffer) __attribute__((always_inline)) {
    if (!left) return;
    ++ahead;
    if (END && next_step == all_steps - 1) {
      const int rest = K - next_step * kWideK;
      ra.load_end(rest, reinterpret_cast<const T*>(castle_weights_zeros), lds0 + buffer);
      rb.load_end(rest, reinterpret_cast<const T*>(castle_weights_zeros), lds0 + buffer + kStage / 2);
    } else {
      ra.load(next.p.lda, lds0 + buffer);
      rb.load(next.p.ldb, lds0 + buffer + kStage / 2);
    }
    if (++next_step == next.from + next.steps) {
      left = at(++next_i, next);
      if (left) start();
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
    OpA::read(l, fa[slot], wm, s, c, g);
    OpB::read(l + kTile * kWideK, fb[slot], wn, s, c, g);
    __builtin_amdgcn_sched_barrier(0);   // these reads, then the products of the fragments before
  };
  arrive();
  read(0, 0);
  for (int i = 0; i == 0 || at(i, unit); ++i) {
    const WeightProduct& p = unit.p;
    const int m0 = unit.m0, n0 = unit.n0;
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
    for (int it = 0; it < unit.steps; ++it) {
#pragma unroll
      for (int s = 0; s < kWideK / 16 - 1; ++s) {
        read(1 - s % 2, s + 1);
        multiply(s % 2);
      }
      arrive();
      done = buffer;
      buffer = kStage - buffer;
      if (it + 1 < unit.steps) request(done);
      read(0, 0);   // (behind the last step of all: what is there, for nothing)
      multiply(1);
    }
    asm volatile("s_nop 15\n\ts_nop 3" ::: "memory");   // the loop may end right behind a product
    __builtin_amdgcn_sched_barrier(0);
    request(done);
    if (unit.slot >= 0) {
      vec<float, 4>* part = reinterpret_cast<vec<float, 4>*>(parts + (int64_t)unit.slot * kPart) + wave * 2048 + lane;
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
template <typename T, bool END> __global__ __launch_bounds__(kWideThreads, 2) void weights_kernel(WeightsArgs a) {
  const int all_steps = (a.R + kWideK - 1) / kWideK, stride = gridDim.x, last = a.whole + a.rest * a.ranges;
  const int first = blockIdx.x % 8 * (stride / 8) + blockIdx.x / 8;   // XCD x takes the x-th eighth of a round
  run_units<T, false, END>([&](int i, Unit& u) __attribute__((always_inline)) {
    const int k = first + i * stride;
    if (k >= last) return false;
    int tile = k;
    u.from = 0;
    u.steps = all_steps;
    u.slot = -1;
    if (k >= a.whole) {
      const int q = (k - a.whole) / a.rest;
      tile = k - q * a.rest;
      u.from = q * a.steps;
      u.steps = min(a.steps, all_steps - u.from);
      if (a.ranges > 1) u.slot = k - a.whole;
    }
    u.p = place(a, tile, u.m0, u.n0);
    return true;
  }, a.R, a.part);
}
// The input gradient too, where its tiles do not fill a round of the card: some workgroups of every XCD have one of its tiles and then a short range of the rows, the others a long range.  Backward pass, us, dx by itself / here: 8192
// rows of 512 through 1408 127 / 116, 12345 of 512 through 1400 183 / 167, 20000 of 256 through 1024 132 / 117; where dx fills its rounds by itself it is behind (16384 of 512 through 1408 200 / 210).
template <typename T, bool END> __global__ __launch_bounds__(kWideThreads, 2) void gradients_kernel(WeightsArgs a) {
  const int xcd = blockIdx.x % 8, j = blockIdx.x / 8, all_steps = (a.R + kWideK - 1) / kWideK;
  const bool has_x = j < a.x_groups;
  if (has_x) {
    run_units<T, true, END>([&](int i, Unit& u) __attribute__((always_inline)) {
      const int t = xcd * a.x_groups + j;
      if (i > 0 || t >= tiles_of(a.x.M, a.x.N)) return false;
      u.p = a.x;
      place_in(a.x, t, u.m0, u.n0);
      u.from = 0;
      u.steps = (a.x_steps + kWideK - 1) / kWideK;
      u.slot = -1;
      return true;
    }, a.x_steps, nullptr);
    __syncthreads();
  }
  run_units<T, false, END>([&](int i, Unit& u) __attribute__((always_inline)) {
    const int others = 32 - a.x_groups, k = has_x ? xcd * a.x_groups + j : xcd * others + j - a.x_groups;   // of the short or of the long ranges
    if (i > 0 || k >= a.rest * (has_x ? a.ranges - a.longs : a.longs)) return false;
    const int q = k / a.rest, tile = k - q * a.rest;
    u.from = has_x ? a.longs * a.long_steps + q * a.steps : q * a.long_steps;
    u.steps = min(has_x ? a.steps : a.long_steps, all_steps - u.from);
    u.slot = a.ranges > 1 ? (has_x ? a.longs * a.rest : 0) + k : -1;
    u.p = place(a, tile, u.m0, u.n0);
    return true;
  }, a.R, a.part);
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
  const WeightProduct p = place(a, a.whole + t, m0, n0);
  const int lane = at & 63, q = at >> 6 & 3, j = at >> 8 & 3, i = at >> 10 & 1, wave = at >> 11;
  const int m = m0 + wave / 2 * 64 + 32 * i + (lane & 31), n = n0 + wave % 2 * 128 + 32 * j + 8 * q + 4 * (lane >> 5);
  if (m < p.M && n < p.N) *reinterpret_cast<vec<T, 4>*>(static_cast<T*>(p.c) + (int64_t)m * p.N + n) = __builtin_convertvector(sum, vec<T, 4>);
}

template <typename Kernel> int launch_kernel(Kernel kernel, PerDeviceOnce& once, int groups, const WeightsArgs& a, hipStream_t stream) {
  bool& configured = once.flag();
  if (!configured) {
    if (hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, kLds) != hipSuccess) return -3;
    configured = true;
  }
  hipLaunchKernelGGL(kernel, dim3(groups), dim3(kWideThreads), kLds, stream, a);
  return hipGetLastError() == hipSuccess ? 0 : -3;
}
template <typename T, bool END> int launch_kernels(const WeightsArgs& a, hipStream_t stream) {
  static PerDeviceOnce once[2];
  if (a.x.c != nullptr) return launch_kernel(&gradients_kernel<T, END>, once[0], kCus, a, stream);
  return launch_kernel(&weights_kernel<T, END>, once[1], std::min((a.whole + a.rest * a.ranges + 7) / 8 * 8, kCus), a, stream);
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
// The input gradient, of M x N over K, in the same launch: cost 1e30 where there is no room for its tiles beside the ranges.  A workgroup that has one goes on to a range that is as much shorter.
WeightsPlan gradients_plan(int R, int M0, int N0, int M1, int N1, int M, int N, int K) {
  WeightsPlan p = {0, 0, 1, 0, 1e30f};
  const int64_t n64 = (int64_t)tiles_of(M0, N0) + tiles_of(M1, N1), x64 = tiles_of(M, N);
  if (n64 > kCus || x64 > kCus * 3 / 4) return p;
  const int n = (int)n64, steps = (R + kWideK - 1) / kWideK, x_steps = (K + kWideK - 1) / kWideK, groups = ((int)x64 + 7) / 8;
  // us a step: 1.9 of ranges, whose rows come from HBM, 1.5 of dx
  int longs = 8 * (32 - groups) / n, shorts = 8 * groups / n;
  if (longs == 0) return p;
  int each = shorts > 0 ? (steps - (int)(longs * (x_steps * 0.79f + 2))) / (longs + shorts) : 0;   // of a short one (2: the change from one to the other)
  if (each <= 0) each = shorts = 0;
  const int most = (steps - shorts * each + longs - 1) / longs;
  longs = std::min(longs, (steps + most - 1) / most);
  const int left = std::max(0, steps - longs * most);   // of the short ones
  shorts = left > 0 ? (left + each - 1) / each : 0;
  p = {0, n, longs + shorts, shorts > 0 ? each : 0, 0, groups, longs, most};
  const int parts = p.ranges > 1 ? n * p.ranges : 0;
  p.cost = 8 + std::max(most * 1.9f, x_steps * 1.5f + (shorts > 0 ? 3 + each * 1.9f : 0)) + 4 + (parts > 0 ? 4 + parts * 0.05f : 0);
  return p;
}
int64_t weights_workspace(const WeightsPlan& p) { return p.ranges > 1 ? (int64_t)p.rest * p.ranges * kPart * 4 : 0; }

int launch_weights(const WeightProduct& first, const WeightProduct& second, const WeightProduct* x, int K, int R, const WeightsPlan& p, int dtype, float* workspace, hipStream_t stream) {
  const WeightsArgs a = {{first, second}, tiles_of(first.M, first.N), R, p.whole, p.rest, p.ranges, p.steps, workspace, x != nullptr ? *x : WeightProduct{}, p.x_groups, K, p.longs, p.long_steps};
  return by_type16(dtype, true, [&](auto t, auto) {
    using T = decltype(t);
    const int rc = R % kWideK == 0 && (x == nullptr || K % kWideK == 0) ? launch_kernels<T, false>(a, stream) : launch_kernels<T, true>(a, stream);
    if (rc == 0 && p.ranges > 1) hipLaunchKernelGGL((weights_join_kernel<T>), dim3(p.rest * (kPart / 1024)), dim3(256), 0, stream, a);
    return rc != 0 ? rc : hipGetLastError() == hipSuccess ? 0 : -3;
  });
}

}  // namespace castle
