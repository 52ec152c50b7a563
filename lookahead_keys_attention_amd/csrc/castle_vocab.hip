// Mean, sum or each of the cross entropies of hidden rows x [R][D] against a vocabulary w [V][D], without the R x V logits z = x w^T in memory:
//
//   loss r = lse r - z[r][target r],  lse r = log sum_v exp z[r][v]              d[r][v] = g r (exp(z[r][v] - lse r) - [v = target r])
//   dx[r] = sum_v d[r][v] w[v]                                                  dw[v] = sum_r d[r][v] x[r]
//
// Forward: tiles of the product x w^T stay in registers, where each wave reduces its 32 ... 128 columns of a row to a maximum and a sum; these are joined by row.
// Backward: the same product again, turned into d on its way to memory in the 16-bit type, for as many columns of the vocabulary at a time as kPieceBytes hold; two products read a
// piece.  Four products in all, where keeping the logits takes three: what it saves is memory, 2 bytes times R V, and the passes over it.
//
// Rows that do not count (target = ignore) are left out at the start: the others are copied together, and what the products cost goes with their number, which the kernels
// read from device memory.  So whatever a row that does not count holds, infinities and NaNs too, goes nowhere.
//
// fp32: the products are those of castle_gemm32.hip, the logits of a piece lie in memory, and kernels over rows do the rest.
#include "castle_tiles.h"
#include "castle_dispatch.h"
#include "castle_gemm.h"
#include "castle_rows.h"
#include "castle_vocab.h"
#include "castle_wide.h"
#include <algorithm>

namespace castle {
namespace {

constexpr int64_t kPieceBytes = (int64_t)1 << 30;
constexpr int kWaves = kThreads / 64;
constexpr int kCountRows = 1024;   // rows of a workgroup that counts
constexpr int kGatherRows = 16;    // rows of a workgroup that copies
constexpr int kLossRows = 16;      // rows of a workgroup that joins maxima and sums

// Where maxima start: a score of -inf has weight 0 behind it wherever it stands, and log2(e) times it is finite.
constexpr float kLeast = -0.5f * __FLT_MAX__;

__host__ __device__ constexpr int64_t up(int64_t n, int64_t to) { return (n + to - 1) / to * to; }

// ---- rows that count -----------------------------------------------------------------------------------------------
struct RowArgs {
  VocabArgs v;
  int* block_counts;   // [R / kCountRows]
  VocabHead* head;
  int32_t* rank;
  void* xc;            // [Rp][Dp]: rows that count, then zero rows up to `zero_to` of them (a multiple of 64, or all)
  int32_t* tc;         // [Rp] their targets, -1 outside of the vocabulary
  float* tl;           // [Rp] logits of the targets: NaN until they are found
  int Dp, zero_all;
  void* loss;          // kEachLoss: zeros for the rows that do not count
};
__device__ __forceinline__ int64_t class_of(const VocabArgs& a, int64_t r) {
  if (a.n == a.R) return a.target[r];
  const uint32_t q = (uint32_t)r / (uint32_t)a.n;   // (rows are fewer than 2^31)
  return a.target[q * a.target_ld + ((uint32_t)r - q * (uint32_t)a.n)];
}
template <int W> __device__ __forceinline__ int sum_over_threads(int v, int* s) {   // s: [W]
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) v += __shfl_xor(v, o);
  if (lane_id() == 0) s[wave_id()] = v;
  __syncthreads();
  v = 0;
#pragma unroll
  for (int w = 0; w < W; ++w) v += s[w];
  __syncthreads();
  return v;
}
__global__ __launch_bounds__(kThreads) void count_rows_kernel(RowArgs a) {
  __shared__ int s[kWaves];
  int n = 0;
  const int64_t first = (int64_t)blockIdx.x * kCountRows;
#pragma unroll
  for (int k = 0; k < kCountRows / kThreads; ++k) {
    const int64_t r = first + k * kThreads + threadIdx.x;
    n += r < a.v.R && class_of(a.v, r) != a.v.ignore;
  }
  n = sum_over_threads<kWaves>(n, s);
  if (threadIdx.x == 0) a.block_counts[blockIdx.x] = n;
}
// FIRST: ranks and targets are formed here, else (backward pass) the ranks are there
template <typename T, bool FIRST> __global__ __launch_bounds__(kThreads) void gather_rows_kernel(RowArgs a) {
  constexpr int V = elem_traits<T>::vec16;
  typedef vec<T, V> vt;
  __shared__ int s[kWaves], s_rank[kGatherRows];
  const int64_t first = (int64_t)blockIdx.x * kGatherRows;
  int all;
  if constexpr (FIRST) {
    const int blocks = (a.v.R + kCountRows - 1) / kCountRows, mine = (int)(first / kCountRows);
    int before = 0, total = 0;
    for (int b = threadIdx.x; b < blocks; b += kThreads) {
      const int n = a.block_counts[b];
      total += n;
      before += b < mine ? n : 0;
    }
    for (int64_t r = (int64_t)mine * kCountRows + threadIdx.x; r < first; r += kThreads) before += class_of(a.v, r) != a.v.ignore;
    before = sum_over_threads<kWaves>(before, s);
    all = sum_over_threads<kWaves>(total, s);
    if (wave_id() == 0) {
      const int64_t r = first + lane_id();
      const bool mine = lane_id() < kGatherRows, there = mine && r < a.v.R;
      const int64_t t = there ? class_of(a.v, r) : a.v.ignore;
      const bool counts = t != a.v.ignore;
      const uint64_t mask = __ballot(counts);
      const int rank = counts ? before + __popcll(mask & ((1ull << lane_id()) - 1)) : -1;
      if (mine) s_rank[lane_id()] = rank;
      if (there) a.rank[r] = rank;
      if (counts) {
        a.tc[rank] = t >= 0 && t < a.v.V ? (int32_t)t : -1;
        a.tl[rank] = NAN;
      }
      if (a.v.reduction == kEachLoss && there && !counts) static_cast<T*>(a.loss)[r] = (T)0.f;
    }
    if (blockIdx.x == 0 && threadIdx.x == 0) *a.head = {all, 1.f / (float)all};
  } else {
    all = a.head->count;
    if (threadIdx.x < kGatherRows) {
      const int64_t r = first + lane_id();
      const int rank = r < a.v.R ? a.rank[r] : -1;
      s_rank[lane_id()] = rank;
      if (rank >= 0) {
        const int64_t t = class_of(a.v, r);
        a.tc[rank] = t >= 0 && t < a.v.V ? (int32_t)t : -1;
      }
    }
  }
  __syncthreads();
  const int pieces = a.Dp / V, have = a.v.D / V;
  const vt none = {};
  const int zero_end = a.zero_all ? a.v.R : (int)up(all, 64);
  for (int k = wave_id(); k < kGatherRows; k += kWaves) {
    const int rank = s_rank[k];
    if (rank >= 0) {
      const T* from = static_cast<const T*>(a.v.x) + (first + k) * a.v.ld_x;
      T* to = static_cast<T*>(a.xc) + (int64_t)rank * a.Dp;
#pragma unroll 4
      for (int i = lane_id(); i < pieces; i += 64) *reinterpret_cast<vt*>(to + i * V) = i < have ? *reinterpret_cast<const vt*>(from + i * V) : none;
    }
    const int64_t r = first + k;   // (the workgroups reach to the next multiple of 64)
    if (r >= all && r < zero_end) {
      T* to = static_cast<T*>(a.xc) + r * a.Dp;
      for (int i = lane_id(); i < pieces; i += 64) *reinterpret_cast<vt*>(to + i * V) = none;
    }
  }
}

// maxima and sums of the P column ranges -> log-sum-exp of a row, its loss; partial sums of the losses, one of each workgroup
struct LossArgs {
  const vec<float, 2>* parts;   // [P][Rp]
  const VocabHead* head;
  const int32_t* rank;
  const float* tl;
  float *lse, *loss_c, *sums;   // loss_c: [Rp] by rank
  void* loss;
  int R, P, reduction;
  int64_t Rp;
};
__global__ __launch_bounds__(kThreads) void row_loss_kernel(LossArgs a) {
  typedef vec<float, 2> v2;
  __shared__ float s_m[kLossRows][kThreads / kLossRows + 1], s_s[kLossRows][kThreads / kLossRows + 1];
  const int c = threadIdx.x % kLossRows, q = threadIdx.x / kLossRows, row = blockIdx.x * kLossRows + c, count = a.head->count;
  float m = kLeast, s = 0.f;
  if (row < count) {
#pragma unroll 8
    for (int p = q; p < a.P; p += kThreads / kLossRows) {
      const v2 x = a.parts[p * a.Rp + row];
      const float mn = fmaxf(m, x[0]);
      s = s * fast_exp2((m - mn) * kLog2e) + x[1] * fast_exp2((x[0] - mn) * kLog2e);
      m = mn;
    }
  }
  s_m[c][q] = m;
  s_s[c][q] = s;
  __syncthreads();
  float loss = 0.f;
  if (q == 0 && row < count) {
    for (int k = 1; k < kThreads / kLossRows; ++k) {
      const float mn = fmaxf(m, s_m[c][k]);
      s = s * fast_exp2((m - mn) * kLog2e) + s_s[c][k] * fast_exp2((s_m[c][k] - mn) * kLog2e);
      m = mn;
    }
    const float lse = m + logf(s);
    a.lse[row] = lse;
    loss = lse - a.tl[row];
    a.loss_c[row] = loss;
  }
  if (threadIdx.x < 64) {
#pragma unroll
    for (int o = 1; o < kLossRows; o <<= 1) loss += __shfl_xor(loss, o);
    if (threadIdx.x == 0) a.sums[blockIdx.x] = loss;
  }
}
template <typename T> __global__ __launch_bounds__(kThreads) void loss_kernel(LossArgs a, int groups) {
  if (a.reduction == kEachLoss) {
    const int64_t r = (int64_t)blockIdx.x * kThreads + threadIdx.x;
    if (r < a.R && a.rank[r] >= 0) static_cast<T*>(a.loss)[r] = (T)a.loss_c[a.rank[r]];
    return;
  }
  __shared__ float s[kWaves];
  float v = 0.f;
  for (int i = threadIdx.x; i < groups; i += kThreads) v += a.sums[i];
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) v += __shfl_xor(v, o);
  if (lane_id() == 0) s[wave_id()] = v;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < kWaves; ++w) v += s[w];
    *static_cast<T*>(a.loss) = (T)(a.reduction == kMeanLoss ? v / (float)a.head->count : v);
  }
}

// Factors of the rows of d.  d lies in the 16-bit type, so the largest factor is brought to 2^14 ... 2^15 by a power of two, 2^shift, which the gradients lose again: softmax
// values down to 2^-29 are then normal numbers of fp16 (without it, a mean over 16384 rows would leave nothing of any below 2^-1), and d stays below 2^15.
struct FactorArgs {
  const void* dloss;
  const VocabHead* head;
  const int32_t *rank, *tc;
  float* factor;   // [Rp] by rank
  int* shift;
  int R, reduction, scaled;
};
template <typename T> __global__ __launch_bounds__(1024) void factor_kernel(FactorArgs a) {
  __shared__ float s[16];
  const bool each = a.reduction == kEachLoss;
  const T* g = static_cast<const T*>(a.dloss);
  float most = 0.f;
  if (each) {
    for (int r = threadIdx.x; r < a.R; r += 1024)
      if (a.rank[r] >= 0) most = fmaxf(most, fabsf((float)g[r]));   // fmaxf drops NaNs
  } else {
    most = fabsf(a.reduction == kMeanLoss ? (float)*g * a.head->inv_count : (float)*g);
  }
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) most = fmaxf(most, __shfl_xor(most, o));
  if (lane_id() == 0) s[wave_id()] = most;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < 16; ++w) most = fmaxf(most, s[w]);
  const int shift = a.scaled && most > 0.f && most <= __FLT_MAX__ ? 15 - __builtin_amdgcn_frexp_expf(most) : 0;
  if (threadIdx.x == 0 && blockIdx.x == 0) *a.shift = shift;
  for (int64_t r = (int64_t)blockIdx.x * 1024 + threadIdx.x; r < a.R; r += (int64_t)gridDim.x * 1024) {
    const int rank = a.rank[r];
    if (rank < 0) continue;
    const float f = each ? (float)g[r] : a.reduction == kMeanLoss ? (float)*g * a.head->inv_count : (float)*g;
    a.factor[rank] = a.tc[rank] >= 0 ? ldexpf(f, shift) : NAN;
  }
}

// steps of each range of a contraction that is split, the last one may have fewer
__host__ __device__ constexpr int steps_of_range(int steps, int splits) { return steps > 0 ? (steps + splits - 1) / splits : 1; }
__host__ __device__ constexpr int ranges(int steps, int splits) { return (steps + steps_of_range(steps, splits) - 1) / steps_of_range(steps, splits); }

// dx[r] = 2^-shift times the sum of its partial results, zeros where it does not count
struct JoinArgs {
  const float* parts;   // [splits][R][D]
  const int32_t* rank;
  const int* shift;
  void* out;
  int splits, D;
  int64_t R;
  const int* count;     // nullptr, or the contraction: there are as many partial results as it has ranges
};
template <typename T> __global__ __launch_bounds__(kThreads) void join_rows_kernel(JoinArgs a) {
  typedef vec<float, 4> v4;
  const int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  const int per = a.D / 4;
  if (i >= a.R * per) return;
  const int64_t r = i / per;
  const int c = (int)(i - r * per) * 4, rank = a.rank == nullptr ? (int)r : a.rank[r];
  v4 v = {0.f, 0.f, 0.f, 0.f};
  if (rank >= 0) {
    const int splits = a.count != nullptr ? ranges((*a.count + kWideK - 1) / kWideK, a.splits) : a.splits;
    const float* p = a.parts + (int64_t)rank * a.D + c;
#pragma unroll 4
    for (int k = 0; k < splits; ++k) v += *reinterpret_cast<const v4*>(p + k * a.R * a.D);
    const int shift = *a.shift;
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = ldexpf(v[e], -shift);
  }
  *reinterpret_cast<vec4_mem<T>*>(static_cast<T*>(a.out) + r * a.D + c) = __builtin_convertvector(v, vec<T, 4>);
}

// ---- products of 16-bit operands ------------------------------------------------------------------------------------
// The frame is that of gemm_wide_kernel (castle_gemm.hip): tiles of the output by workgroups of eight waves, steps of 64 of the contraction straight from memory to LDS into
// two or three buffers, requested over the end of a tile.  What differs: sizes that are read from device memory, contractions of any length (d and the copied rows are padded with
// zeros, and behind the end of w's rows or of a row of it what is there is read again), and what becomes of a tile:
enum { kStats = 0, kGrad = 1, kRowGrad = 2, kWeightGrad = 3 };
struct ProductArgs {
  const void *a, *b;
  int64_t lda, ldb;
  int M, N, K;             // kWeightGrad: K is an upper bound, else M
  const int* count;        // rows that count
  int splits;              // ranges of the contraction, at most
  // kStats
  vec<float, 2>* parts;
  float* tl;
  int64_t Rp;
  // kStats, kGrad
  const int32_t* tc;
  int first;               // column of the vocabulary that n = 0 is
  // kGrad: d, rows of ldc; rows behind the last up to a multiple of 64 and columns N ... ldc - 1 are zero
  const float *lse, *factor;
  void* c;
  int64_t ldc;
  // kRowGrad: partial results [splits][part_rows][N], added to those that are there; kWeightGrad: c, or partial results [splits][M][N] where there are several
  float* out;
  int64_t part_rows;
  int add;
  const int* shift;
};

// d lies in blocks of 64 x 64, whole rows of blocks one behind the other: a step of either product that reads it fetches pieces of 8 KB.  (Rows of d as they are: 128 bytes here and
// there, 64 KB and more apart; dx of 16384 rows over 32000 503 us, dweight 468.)
constexpr int kBlock = 64;
template <typename T, bool KC, int FREE> struct BlockOperand : WideOperand<T, KC, FREE> {
  typedef WideOperand<T, KC, FREE> W;
  // p: [row of blocks][ldc / 64][64][64]
  __device__ __forceinline__ void start(const T* p, int64_t ldc, int free0, int free_end, int k0) {
    const int lane = lane_id(), first = wave_id() * W::N;
    W::left = free_end - free0;
    W::at = KC ? p + free0 * ldc + k0 * kBlock : p + k0 * ldc + free0 * kBlock;
#pragma unroll
    for (int q = 0; q < W::N; ++q) {
      if constexpr (KC) {
        const int row = 8 * (first + q) + (lane >> 3), piece = (lane & 7) ^ (row >> 1 & 7), there = min(row, W::left - 1);
        W::off[q] = 2 * (uint32_t)(there / kBlock * kBlock * (int)ldc + there % kBlock * kBlock + 8 * piece);
      } else {
        constexpr int PIECES = FREE / 8, ROWS = 64 / PIECES;
        const int k = ROWS * (first + q) + lane / PIECES, p = lane % PIECES ^ 4 * (k & 3), piece = 8 * p < W::left ? p : 0;
        W::off[q] = 2 * (uint32_t)(piece / 8 * kBlock * kBlock + k * kBlock + 8 * (piece % 8));
      }
    }
  }
  __device__ __forceinline__ void load(int64_t ldc, uint32_t lds) {
#pragma unroll
    for (int q = 0; q < W::N; ++q) load_to_lds(W::at, W::off[q], lds + 1024 * (wave_id() * W::N + q));
    W::at += kBlock * (KC ? (int64_t)kBlock : ldc);
  }
};

// Eight waves over BM x BN: four by two of them for 256 rows, else two by four.
template <int MODE, int BM, int BN> struct Shape {
  static constexpr int WM = BM == 256 ? 4 : 2, WN = 8 / WM, FM = BM / 32 / WM, FN = BN / 32 / WN;
  static constexpr bool kTurn = MODE == kGrad || MODE == kWeightGrad;   // a tile goes through LDS to whole rows, 4 KB of each wave
  static constexpr int kStage = (BM + BN) * kWideK * 2, kTurnBytes = kTurn ? 4096 * 8 : 0;
  static constexpr int kFit = (kMaxLds - kTurnBytes) / kStage, kStages = kFit < 3 ? kFit : 3;
  static constexpr int kLoads = kStage / 1024 / 8, kLds = kStages * kStage + kTurnBytes;
  static constexpr int kStores = MODE == kStats ? FM : MODE == kRowGrad ? 4 * FM * FN : 2 * FM * FN;   // of a wave and tile (kWeightGrad: partial results are twice as many)
  static_assert(kStages >= 2 && FM >= 1 && FN >= 1, "");
};
extern __shared__ __attribute__((aligned(16))) unsigned char castle_vocab_lds[];

template <typename T, int MODE, int BM, int BN> __global__ __launch_bounds__(kWideThreads, 2) void vocab_product_kernel(ProductArgs a) {
  typedef Shape<MODE, BM, BN> S;
  constexpr bool AK = MODE != kWeightGrad, BKC = MODE == kStats || MODE == kGrad;
  typedef std::conditional_t<MODE == kRowGrad || MODE == kWeightGrad, BlockOperand<T, AK, BM>, WideOperand<T, AK, BM>> OpA;
  typedef WideOperand<T, BKC, BN> OpB;
  typedef vec<T, 8> vt;
  const int lane = lane_id(), wave = wave_id(), c = lane & 31, g = lane >> 5;
  const int count = __builtin_amdgcn_readfirstlane(*a.count), M = MODE == kWeightGrad ? a.M : min(a.M, count), K = MODE == kWeightGrad ? (int)up(min(a.K, count), kWideK) : a.K;
  const int tiles_m = (M + BM - 1) / BM, tiles_n = (a.N + BN - 1) / BN, tiles = tiles_m * tiles_n;
  if (tiles == 0) return;
  // Items are tiles for each range of the contraction; XCD x takes the x-th eighth of them.  Tiles in the order of an XCD's L2: all rows of a band of columns, then those of the next.
  constexpr int kBand = 2048 / BN;
  const int all_steps = (K + kWideK - 1) / kWideK, per_range = steps_of_range(all_steps, a.splits);
  const int items = tiles * max(1, ranges(all_steps, a.splits));
  // The place of an item, moved on by additions: divisions by the sizes took a tenth of what 16384 x 32000 logits of 512 take.
  struct Walk { int band, rest, range; };   // rest: tile of the band
  const int bands = (tiles_n + kBand - 1) / kBand;
  auto advance = [&](Walk& w, int by) __attribute__((always_inline)) {
    w.rest += by;
    while (true) {
      const int size = tiles_m * min(kBand, tiles_n - w.band * kBand);
      if (w.rest < size) break;
      w.rest -= size;
      if (++w.band == bands) {
        w.band = 0;
        ++w.range;
      }
    }
  };
  struct Item { int m0, n0, range, k0, steps; };
  auto item_at = [&](const Walk& w) __attribute__((always_inline)) {
    const int width = min(kBand, tiles_n - w.band * kBand), m = width == kBand ? w.rest / kBand : w.rest / width;
    return Item{m * BM, (w.band * kBand + w.rest - m * width) * BN, w.range, w.range * per_range * kWideK, min(per_range, all_steps - w.range * per_range)};
  };
  const int share = (items + 7) / 8, begin = blockIdx.x % 8 * share, last = min(items, begin + share), stride = gridDim.x / 8;
  const int wm = wave / S::WN * 32 * S::FM, wn = wave % S::WN * 32 * S::FN;
  int item = begin + blockIdx.x / 8;
  if (item >= last) return;
  const bool any = all_steps > 0;
  const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) unsigned char*)castle_vocab_lds;
  // the step that is requested next runs ahead of the one that is multiplied, into the next item
  OpA ra;
  OpB rb;
  Walk at = {0, 0, 0};
  advance(at, item);
  Walk next_at = at;
  int next_item = item, next_steps = 0, next_k = 0, ahead = 0;   // ahead: steps requested and not waited for
  auto start = [&]() __attribute__((always_inline)) {
    const Item t = item_at(next_at);
    next_steps = t.steps;
    next_k = t.k0;
    ra.start(static_cast<const T*>(a.a), a.lda, t.m0, M, t.k0);
    rb.start(static_cast<const T*>(a.b), a.ldb, t.n0, a.N, t.k0);
  };
  auto request = [&](int buffer) __attribute__((always_inline)) {
    if (next_item >= last) return;
    ++ahead;
    if constexpr (MODE != kWeightGrad)
      if (next_k + kWideK > K) rb.place((int)a.ldb, K - next_k);
    ra.load(a.lda, lds0 + buffer);
    rb.load(a.ldb, lds0 + buffer + BM * kWideK * 2);
    next_k += kWideK;
    if (--next_steps == 0) {
      next_item += stride;
      if (next_item < last) {
        advance(next_at, stride);
        start();
      }
    }
  };
  if (any) {
    start();
    request(0);
    request(S::kStage);
    if constexpr (S::kStages == 3) request(2 * S::kStage);
  }
  // The step behind the current one is in LDS, from every wave, and all have read the current one.  Waits are for all but the last so many requests; the stores of a
  // tile inside the output, kStores at least, come behind those and are not waited for (`stored`).
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
    const T* la = reinterpret_cast<const T*>(castle_vocab_lds + buffer);
    OpA::read(la, fa[slot], wm, s, c, g);
    OpB::read(la + BM * kWideK, fb[slot], wn, s, c, g);
    __builtin_amdgcn_sched_barrier(0);   // these reads, then the products of the fragments before
  };
  if (any) arrive();
  while (item < last) {
    const auto [m0, n0, range, k0, steps] = item_at(at);
    // What the end of a tile needs of its rows: requested here, there behind the last wait for operands, and the next operands only behind that (the wait for these would
    // include them).
    float l[S::FM], f[S::FM];
    int t[S::FM];
    auto fetch_rows = [&]() __attribute__((always_inline)) {
#pragma unroll
      for (int i = 0; i < S::FM; ++i) {
        const int m = min(m0 + wm + 32 * i + c, M - 1);
        t[i] = a.tc[m];
        if constexpr (MODE == kGrad) {
          l[i] = a.lse[m];
          f[i] = a.factor[m];
        }
      }
    };
    auto rows_are_there = [&]() __attribute__((always_inline)) {
#pragma unroll
      for (int i = 0; i < S::FM; ++i) {
        asm volatile("" : "+v"(t[i]));
        if constexpr (MODE == kGrad) asm volatile("" : "+v"(l[i]), "+v"(f[i]));
      }
    };
    constexpr bool ROWS = MODE == kStats || MODE == kGrad;
    if constexpr (ROWS) fetch_rows();
    if (any) read(0, 0);
    int done = 0;   // buffer of the step that ends
    acc_t acc[S::FM][S::FN];   // [n rows, m lanes]
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
    if constexpr (ROWS) rows_are_there();
    if (any) request(done);
    item += stride;
    if (item < last) advance(at, stride);
    const bool inside = m0 + BM <= M && n0 + BN <= a.N;
    if constexpr (MODE == kStats) {
      // this wave's columns of the row of lane c: 16 FN of them here, as many in lane c + 32
      const int here = n0 + wn + 4 * g;   // column of element (j, r) of this lane, less 32 j + acc_row(r, 0)
#pragma unroll
      for (int i = 0; i < S::FM; ++i) {
        const int m = m0 + wm + 32 * i + c;
        t[i] -= here;
        acc_t z[S::FN];
        const int end = n0 + BN > a.N ? a.N - here : 32 * S::FN;   // columns of this lane that are there
#pragma unroll
        for (int j = 0; j < S::FN; ++j) z[j] = acc[i][j];
        if (n0 + BN > a.N) {
#pragma unroll
          for (int j = 0; j < S::FN; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) z[j][r] = 32 * j + acc_row(r, 0) < end ? z[j][r] : -INFINITY;
        }
        const bool mine = m < M && t[i] >= 0 && t[i] < 32 * S::FN && (t[i] & 4) == 0;
        if (__ballot(mine) != 0) {
          float zt = 0.f;
#pragma unroll
          for (int j = 0; j < S::FN; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) zt = t[i] == 32 * j + acc_row(r, 0) ? z[j][r] : zt;
          if (mine) a.tl[m] = zt;
        }
        float most = kLeast;
#pragma unroll
        for (int j = 0; j < S::FN; ++j)
#pragma unroll
          for (int r = 0; r < 16; r += 2) most = fmaxf(fmaxf(most, z[j][r]), z[j][r + 1]);   // fmaxf drops NaNs
        most = fmaxf(most, __shfl_xor(most, 32));
        const float shift = most * kLog2e;
        float sum[4] = {};
#pragma unroll
        for (int j = 0; j < S::FN; ++j)
#pragma unroll
          for (int r = 0; r < 16; ++r) sum[r % 4] += fast_exp2(__builtin_fmaf(z[j][r], kLog2e, -shift));
        float s = (sum[0] + sum[1]) + (sum[2] + sum[3]);
        s += __shfl_xor(s, 32);
        if (g == 0 && m < M) a.parts[(int64_t)(n0 / BN * S::WN + wave % S::WN) * a.Rp + m] = vec<float, 2>{most, s};
        __builtin_amdgcn_sched_barrier(0);
      }
      stored = inside;
    } else if constexpr (MODE == kRowGrad) {
      float* out = a.out + (int64_t)range * a.part_rows * a.N;
#pragma unroll
      for (int i = 0; i < S::FM; ++i) {
        const int m = m0 + wm + 32 * i + c;
        float* row = out + (int64_t)m * a.N + n0 + wn + 4 * g;
#pragma unroll
        for (int j = 0; j < S::FN; ++j)
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            if (m >= M || n0 + wn + 32 * j + 8 * q + 4 * g >= a.N) continue;
            vec<float, 4>* p = reinterpret_cast<vec<float, 4>*>(row + 32 * j + 8 * q);
            vec<float, 4> v = pack4<float>(acc[i][j], q);
            if (a.add) v += *p;
            *p = v;
          }
        __builtin_amdgcn_sched_barrier(0);
      }
      stored = inside && !a.add;
    } else if (MODE == kWeightGrad && a.splits > 1) {
      float* out = a.out + (int64_t)range * a.M * a.N;
#pragma unroll
      for (int i = 0; i < S::FM; ++i) {
        const int m = m0 + wm + 32 * i + c;
        float* row = out + (int64_t)m * a.N + n0 + wn + 4 * g;
#pragma unroll
        for (int j = 0; j < S::FN; ++j)
#pragma unroll
          for (int q = 0; q < 4; ++q)
            if (m < M && n0 + wn + 32 * j + 8 * q + 4 * g < a.N) *reinterpret_cast<vec<float, 4>*>(row + 32 * j + 8 * q) = pack4<float>(acc[i][j], q);
        __builtin_amdgcn_sched_barrier(0);
      }
      stored = inside;
    } else {
      // to whole rows through LDS, 32 rows of up to 64 columns at a time, each wave in a part of its own; pieces placed as in the operands
      T* turn = reinterpret_cast<T*>(castle_vocab_lds + S::kStages * S::kStage + wave * 4096);
      constexpr int FJ = S::FN < 2 ? 1 : 2, CP = 4 * FJ, RP = 64 / CP;   // CP: pieces of a row; RP: rows of a store
      const int shift = MODE == kWeightGrad ? __builtin_amdgcn_readfirstlane(*a.shift) : 0;
      const int row_end = MODE == kGrad ? min((int)up(count, 64), (int)a.Rp) : M;
#pragma unroll
      for (int i = 0; i < S::FM; ++i) {
        acc_t z[S::FN];
#pragma unroll
        for (int j = 0; j < S::FN; ++j) z[j] = acc[i][j];
        if constexpr (MODE == kGrad) {
          const float shift = l[i] * kLog2e;
          t[i] -= a.first + n0 + wn + 4 * g;
          // g exp(z - lse), a factor that is not negative in the exponent; less the factor at the target
          auto form = [&](auto target) __attribute__((always_inline)) {
            const float up = __builtin_amdgcn_logf(f[i]) - shift;
#pragma unroll
            for (int j = 0; j < S::FN; ++j)
#pragma unroll
              for (int r = 0; r < 16; ++r) {
                float p = fast_exp2(__builtin_fmaf(z[j][r], kLog2e, up));
                if constexpr (decltype(target)::value) p -= t[i] == 32 * j + acc_row(r, 0) ? f[i] : 0.f;
                z[j][r] = p;
              }
          };
          auto form_any = [&]() __attribute__((always_inline)) {
            const int end = m0 + wm + 32 * i + c < M ? a.N - n0 - wn - 4 * g : 0;
#pragma unroll
            for (int j = 0; j < S::FN; ++j)
#pragma unroll
              for (int r = 0; r < 16; ++r) {
                const int n = 32 * j + acc_row(r, 0);
                const float p = fast_exp2(__builtin_fmaf(z[j][r], kLog2e, -shift)) - (t[i] == n ? 1.f : 0.f);
                z[j][r] = n < end ? p * f[i] : 0.f;
              }
          };
          if (!inside || __ballot(f[i] < 0.f) != 0) form_any();
          else if (__ballot(t[i] >= 0 && t[i] < 32 * S::FN) != 0) form(std::true_type());
          else form(std::false_type());
        } else {
#pragma unroll
          for (int j = 0; j < S::FN; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) z[j][r] = ldexpf(z[j][r], -shift);
        }
#pragma unroll
        for (int h = 0; h < S::FN / FJ; ++h) {
          __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
          __builtin_amdgcn_wave_barrier();
#pragma unroll
          for (int j = 0; j < FJ; ++j)
#pragma unroll
            for (int q = 0; q < 4; ++q) st4<T>(turn + c * 8 * CP + 8 * ((4 * j + q) ^ (c >> 1 & (CP - 1))) + 4 * g, pack4<T>(z[FJ * h + j], q));
          __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
          __builtin_amdgcn_wave_barrier();
#pragma unroll
          for (int k = 0; k < 32 / RP; ++k) {
            const int row = RP * k + lane / CP, piece = lane % CP, mm = m0 + wm + 32 * i + row, n = n0 + wn + 32 * FJ * h + 8 * piece;
            const vt v = *reinterpret_cast<const vt*>(turn + row * 8 * CP + 8 * (piece ^ (row >> 1 & (CP - 1))));
            T* to = static_cast<T*>(a.c) + (MODE == kGrad ? (int64_t)(mm / kBlock * kBlock) * a.ldc + n / kBlock * (kBlock * kBlock) + mm % kBlock * kBlock + n % kBlock
                                                          : (int64_t)mm * a.ldc + n);
            if (mm < row_end && n < (MODE == kGrad ? (int)a.ldc : a.N)) *reinterpret_cast<vt*>(to) = v;
          }
        }
      }
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      stored = inside;
    }
  }
}

template <typename T, int MODE, int BM, int BN> int launch_product_t(const ProductArgs& a, hipStream_t stream) {
  typedef Shape<MODE, BM, BN> S;
  static PerDeviceOnce once;
  bool& configured = once.flag();
  if (!configured) {
    if (hipFuncSetAttribute(reinterpret_cast<const void*>(&vocab_product_kernel<T, MODE, BM, BN>), hipFuncAttributeMaxDynamicSharedMemorySize, S::kLds) != hipSuccess) return -3;
    configured = true;
  }
  const int64_t items = up(a.M, BM) / BM * (up(a.N, BN) / BN) * a.splits;
  hipLaunchKernelGGL((vocab_product_kernel<T, MODE, BM, BN>), dim3((unsigned)std::min<int64_t>(up(items, 8), 256)), dim3(kWideThreads), S::kLds, stream, a);
  return hipGetLastError() == hipSuccess ? 0 : -3;
}
// rows and columns of a workgroup's tile
struct Tile { int rows, columns; };
Tile logits_tile(int R) { return {R <= 64 ? 64 : 256, 256}; }
Tile row_grad_tile(int R, int D) { return {R <= 64 ? 64 : 256, D <= 128 ? 128 : 256}; }
Tile weight_grad_tile(int D) { return {256, D <= 128 ? 128 : 256}; }
template <typename T, int MODE> int launch_logits(const ProductArgs& a, hipStream_t stream) {
  return logits_tile(a.M).rows == 64 ? launch_product_t<T, MODE, 64, 256>(a, stream) : launch_product_t<T, MODE, 256, 256>(a, stream);
}
template <typename T> int launch_row_grad(const ProductArgs& a, hipStream_t stream) {
  const Tile t = row_grad_tile(a.M, a.N);
  if (t.rows == 64) return t.columns == 128 ? launch_product_t<T, kRowGrad, 64, 128>(a, stream) : launch_product_t<T, kRowGrad, 64, 256>(a, stream);
  return t.columns == 128 ? launch_product_t<T, kRowGrad, 256, 128>(a, stream) : launch_product_t<T, kRowGrad, 256, 256>(a, stream);
}
template <typename T> int launch_weight_grad(const ProductArgs& a, hipStream_t stream) {
  return weight_grad_tile(a.N).columns == 128 ? launch_product_t<T, kWeightGrad, 256, 128>(a, stream) : launch_product_t<T, kWeightGrad, 256, 256>(a, stream);
}

// ---- sizes ----------------------------------------------------------------------------------------------------------
int pieces_of_row(int R) { return (R + kLossRows - 1) / kLossRows; }
struct Plan {
  int64_t Rp;              // rows, a multiple of 64
  int Dp;                  // width of a copied row
  int P;                   // column ranges of a row's maxima and sums
  int columns, pieces;     // of the vocabulary at a time
  int64_t ldc;             // of d (fp32: of the logits)
  int row_splits, weight_splits;
};
int64_t tiles(int64_t m, int64_t n, Tile t) { return up(m, t.rows) / t.rows * (up(n, t.columns) / t.columns); }
// Ranges of a contraction of `steps` for m x n outputs, from what it takes roughly (us): 1.5 a step and 5 an end for each of the items of the fullest CU, and for several ranges their partial
// results, written and read at 4 TB/s.
int splits_for(int64_t m, int64_t n, Tile t, int64_t steps) {
  int best = 1;
  double best_cost = 1e30;
  for (int s = 1; s <= 128 && s <= std::max<int64_t>(1, steps / 2); ++s) {
    const double cost = (tiles(m, n, t) * s + 255) / 256 * (1.5 * steps_of_range((int)steps, s) + 5) + (s > 1 ? 8e-6 / 4 * s * m * n : 0);
    if (cost < best_cost) {
      best_cost = cost;
      best = s;
    }
  }
  return best;
}
Plan plan(const VocabArgs& a, int es) {
  Plan p = {};
  p.Rp = up(a.R, 64);
  p.Dp = es == 2 ? (int)up(a.D, kWideK) : a.D;
  const int64_t fit = kPieceBytes / (p.Rp * es) / 256 * 256, width = up(a.V, 64);
  p.pieces = (int)((width + std::max<int64_t>(256, fit) - 1) / std::max<int64_t>(256, fit));
  p.columns = (int)up((a.V + p.pieces - 1) / p.pieces, 256);
  p.pieces = (a.V + p.columns - 1) / p.columns;
  p.ldc = std::min<int64_t>(p.columns, width);
  if (es == 2) {
    const Tile t = logits_tile(a.R);
    p.P = (int)(up(a.V, t.columns) / t.columns * (t.rows == 256 ? 2 : 4));
  } else {
    p.P = p.pieces;
  }
  p.row_splits = splits_for(a.R, a.D, row_grad_tile(a.R, a.D), p.ldc / kWideK);
  p.weight_splits = splits_for(p.ldc, a.D, weight_grad_tile(a.D), p.Rp / kWideK);
  return p;
}
// what the fp32 products of `bytes(columns)` need: of a whole piece of the vocabulary, and of the last one
template <typename F> int64_t products32(const VocabArgs& a, const Plan& p, F&& bytes) { return std::max(bytes(std::min(a.V, p.columns)), bytes(a.V - (p.pieces - 1) * p.columns)); }
struct Carve {
  char* at;
  int64_t used = 0;
  template <typename U> U* take(int64_t n) {
    U* p = reinterpret_cast<U*>(at + used);
    used += up(n * (int64_t)sizeof(U), 256);
    return p;
  }
};
struct Fwd {
  int* block_counts;
  char* xc;
  int32_t* tc;
  float *tl, *loss_c, *sums;
  vec<float, 2>* parts;
  char* logits;
  Fwd(const VocabArgs& a, const Plan& p, int es, Carve& c) {
    block_counts = c.take<int>(up(a.R, kCountRows) / kCountRows);
    xc = c.take<char>(p.Rp * p.Dp * es);
    tc = c.take<int32_t>(p.Rp);
    tl = c.take<float>(p.Rp);
    loss_c = c.take<float>(p.Rp);
    sums = c.take<float>(pieces_of_row(a.R));
    parts = c.take<vec<float, 2>>(p.P * p.Rp);
    logits = c.take<char>(es == 4 ? a.R * p.ldc * 4 : 0);
  }
};
struct Bwd {
  char* xc;
  int32_t* tc;
  float* factor;
  int* shift;
  char* d;
  float *row_parts, *weight_parts;
  char* products;
  Bwd(const VocabArgs& a, const Plan& p, int es, bool need_x, bool need_w, Carve& c) {
    xc = c.take<char>(p.Rp * p.Dp * es);
    tc = c.take<int32_t>(p.Rp);
    factor = c.take<float>(p.Rp);
    shift = c.take<int>(1);
    d = c.take<char>(p.Rp * p.ldc * es);
    row_parts = c.take<float>(need_x ? (int64_t)(es == 2 ? p.row_splits : p.pieces > 1 ? 2 : 1) * a.R * a.D : 0);
    weight_parts = c.take<float>(need_w && es == 2 && p.weight_splits > 1 ? p.weight_splits * p.ldc * a.D : 0);
    products = c.take<char>(es == 2 ? 0 : products32(a, p, [&](int n) {
      return std::max(gemm_workspace(a.R, a.D, n, 4, false), gemm_workspace(n, a.D, a.R, 4, false));
    }));
  }
};
struct State {
  VocabHead* head;
  int32_t* rank;
  float* lse;
  State(int64_t R, Carve& c) {
    head = c.take<VocabHead>(1);
    rank = c.take<int32_t>(R);
    lse = c.take<float>(R);
  }
};
int launched() { return hipGetLastError() == hipSuccess ? 0 : -3; }
template <bool FIRST> int launch_gather(const RowArgs& a, int dtype, hipStream_t stream) {
  return by_tensor_type(dtype, [&](auto t) {
    using T = decltype(t);
    hipLaunchKernelGGL((gather_rows_kernel<T, FIRST>), dim3((unsigned)(up(a.v.R, 64) / kGatherRows)), dim3(kThreads), 0, stream, a);
    return launched();
  });
}

// ---- fp32: logits of a piece in memory -------------------------------------------------------------------------------
struct Rows32 {
  float* z;                // [R][ld]
  int64_t ld, Rp;
  int columns, first;      // of the vocabulary
  const int* count;
  const int32_t* tc;
  float* tl;
  vec<float, 2>* parts;    // of this piece, by rank
  const float *lse, *factor;
};
// a wave to a row
__global__ __launch_bounds__(kThreads) void row_stats32_kernel(Rows32 a) {
  typedef vec<float, 4> v4;
  const int row = blockIdx.x * kWaves + wave_id(), lane = lane_id();
  if (row >= *a.count) return;
  const float* z = a.z + row * a.ld;
  float m = kLeast, s = 0.f;
  for (int i = lane * 4; i < a.columns; i += 256) {
    v4 v = *reinterpret_cast<const v4*>(z + i);   // (rows are padded to whole pieces)
    float mn = m;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (i + e >= a.columns) v[e] = -INFINITY;
      mn = fmaxf(mn, v[e]);
    }
    s *= fast_exp2((m - mn) * kLog2e);
#pragma unroll
    for (int e = 0; e < 4; ++e) s += fast_exp2((v[e] - mn) * kLog2e);
    m = mn;
  }
  float M = m;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) M = fmaxf(M, __shfl_xor(M, o));
  s *= fast_exp2((m - M) * kLog2e);
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) s += __shfl_xor(s, o);
  const int t = a.tc[row] - a.first;
  if (lane == 0) {
    a.parts[row] = vec<float, 2>{M, s};
    if (a.tc[row] >= 0 && t >= 0 && t < a.columns) a.tl[row] = z[t];
  }
}
// z -> d in place; zeros in the rows behind the last
__global__ __launch_bounds__(kThreads) void row_grad32_kernel(Rows32 a, int R) {
  typedef vec<float, 4> v4;
  const int row = blockIdx.x * kWaves + wave_id(), lane = lane_id();
  if (row >= R) return;
  const bool counts = row < *a.count;
  float* z = a.z + row * a.ld;
  const float l = counts ? a.lse[row] : 0.f, f = counts ? a.factor[row] : 0.f;
  const int t = counts ? a.tc[row] - a.first : -1;
  for (int i = lane * 4; i < a.columns; i += 256) {
    v4 v = *reinterpret_cast<const v4*>(z + i);
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = counts && i + e < a.columns ? f * (fast_exp2((v[e] - l) * kLog2e) - (t == i + e ? 1.f : 0.f)) : 0.f;
    *reinterpret_cast<v4*>(z + i) = v;
  }
}
GemmArgs product32(const void* a, int64_t lda, const void* b, int64_t ldb, void* c, int64_t ldc, int M, int N, int K, bool whole = false) {
  GemmArgs g = {};
  g.a = a;
  g.b = b;
  g.c = c;
  g.M = M;
  g.N = N;
  g.K = K;
  g.lda = lda;
  g.ldb = ldb;
  g.ldc = ldc;
  g.epilogue = kGemmPlain;
  g.whole = whole;
  return g;
}

}  // namespace

int64_t vocab_state_bytes(int64_t R) {
  Carve c = {nullptr};
  State(R, c);
  return c.used;
}
int64_t vocab_fwd_bytes(const VocabArgs& a, int es) {
  Carve c = {nullptr};
  Fwd(a, plan(a, es), es, c);
  return c.used;
}
int64_t vocab_bwd_bytes(const VocabArgs& a, int es, bool need_x, bool need_w) {
  Carve c = {nullptr};
  Bwd(a, plan(a, es), es, need_x, need_w, c);
  return c.used;
}

int launch_vocab_fwd(const VocabArgs& a, int dtype, void* loss, void* state, void* workspace, hipStream_t stream) {
  const int es = dtype == 0 ? 4 : 2;
  const Plan p = plan(a, es);
  Carve cs = {static_cast<char*>(state)}, cw = {static_cast<char*>(workspace)};
  const State s(a.R, cs);
  const Fwd f(a, p, es, cw);
  const RowArgs rows = {a, f.block_counts, s.head, s.rank, f.xc, f.tc, f.tl, p.Dp, es == 4, loss};
  hipLaunchKernelGGL(count_rows_kernel, dim3((unsigned)(up(a.R, kCountRows) / kCountRows)), dim3(kThreads), 0, stream, rows);
  int rc = launch_gather<true>(rows, dtype, stream);
  if (rc != 0) return rc;
  if (es == 2) {
    ProductArgs g = {};
    g.a = f.xc;
    g.b = a.w;
    g.lda = p.Dp;
    g.ldb = a.ld_w;
    g.M = a.R;
    g.N = a.V;
    g.K = a.D;
    g.count = &s.head->count;
    g.splits = 1;
    g.parts = f.parts;
    g.tl = f.tl;
    g.Rp = p.Rp;
    g.tc = f.tc;
    rc = by_type16(dtype, true, [&](auto t, auto) { return launch_logits<decltype(t), kStats>(g, stream); });
    if (rc != 0) return rc;
  } else {
    for (int i = 0; i < p.pieces; ++i) {
      const int v0 = i * p.columns, n = std::min(p.columns, a.V - v0);
      rc = launch_gemm(product32(f.xc, p.Dp, static_cast<const float*>(a.w) + v0 * a.ld_w, a.ld_w, f.logits, p.ldc, a.R, n, a.D, true), true, true, 0, nullptr, stream);
      if (rc != 0) return rc;
      const Rows32 r = {reinterpret_cast<float*>(f.logits), p.ldc, p.Rp, n, v0, &s.head->count, f.tc, f.tl, f.parts + i * p.Rp, nullptr, nullptr};
      hipLaunchKernelGGL(row_stats32_kernel, dim3((a.R + kWaves - 1) / kWaves), dim3(kThreads), 0, stream, r);
      if (launched() != 0) return -3;
    }
  }
  const int groups = pieces_of_row(a.R);
  const LossArgs l = {f.parts, s.head, s.rank, f.tl, s.lse, f.loss_c, f.sums, loss, a.R, p.P, a.reduction, p.Rp};
  hipLaunchKernelGGL(row_loss_kernel, dim3(groups), dim3(kThreads), 0, stream, l);
  return by_tensor_type(dtype, [&](auto t) {
    hipLaunchKernelGGL((loss_kernel<decltype(t)>), dim3(a.reduction == kEachLoss ? (unsigned)(up(a.R, kThreads) / kThreads) : 1), dim3(kThreads), 0, stream, l, groups);
    return launched();
  });
}

int launch_vocab_bwd(const VocabArgs& a, int dtype, const void* dloss, const void* state, void* dx, void* dw, void* workspace, hipStream_t stream) {
  const int es = dtype == 0 ? 4 : 2;
  const Plan p = plan(a, es);
  Carve cs = {static_cast<char*>(const_cast<void*>(state))}, cw = {static_cast<char*>(workspace)};
  const State s(a.R, cs);
  const Bwd b(a, p, es, dx != nullptr, dw != nullptr, cw);
  const RowArgs rows = {a, nullptr, s.head, s.rank, b.xc, b.tc, nullptr, p.Dp, es == 4, nullptr};
  int rc = launch_gather<false>(rows, dtype, stream);
  if (rc != 0) return rc;
  const FactorArgs fa = {dloss, s.head, s.rank, b.tc, b.factor, b.shift, a.R, a.reduction, es == 2};
  rc = by_tensor_type(dtype, [&](auto t) {
    hipLaunchKernelGGL((factor_kernel<decltype(t)>), dim3(std::min<unsigned>(64, (unsigned)(up(a.R, 1024) / 1024))), dim3(1024), 0, stream, fa);
    return launched();
  });
  if (rc != 0) return rc;
  for (int i = 0; i < p.pieces && es == 2; ++i) {
    const int v0 = i * p.columns, n = std::min(p.columns, a.V - v0);
    const char* w = static_cast<const char*>(a.w) + v0 * a.ld_w * es;
    ProductArgs g = {};
    g.a = b.xc;
    g.b = w;
    g.lda = p.Dp;
    g.ldb = a.ld_w;
    g.M = a.R;
    g.N = n;
    g.K = a.D;
    g.count = &s.head->count;
    g.splits = 1;
    g.Rp = p.Rp;
    g.tc = b.tc;
    g.first = v0;
    g.lse = s.lse;
    g.factor = b.factor;
    g.c = b.d;
    g.ldc = p.ldc;
    g.shift = b.shift;
    ProductArgs gx = g, gw = g;
    gx.a = b.d;
    gx.lda = p.ldc;
    gx.N = a.D;
    gx.K = n;
    gx.splits = p.row_splits;
    gx.out = b.row_parts;
    gx.part_rows = a.R;
    gx.add = i > 0;
    gw.a = b.d;
    gw.lda = p.ldc;
    gw.b = b.xc;
    gw.ldb = p.Dp;
    gw.M = n;
    gw.N = a.D;
    gw.K = a.R;
    gw.splits = p.weight_splits;
    gw.c = static_cast<char*>(dw) + (int64_t)v0 * a.D * es;
    gw.ldc = a.D;
    gw.out = b.weight_parts;
    rc = by_type16(dtype, true, [&](auto t, auto) {
      using T = decltype(t);
      int e = launch_logits<T, kGrad>(g, stream);
      if (e == 0 && dx != nullptr) e = launch_row_grad<T>(gx, stream);
      if (e == 0 && dw != nullptr) e = launch_weight_grad<T>(gw, stream);
      if (e == 0 && dw != nullptr && gw.splits > 1) {
        const JoinArgs j = {b.weight_parts, nullptr, b.shift, gw.c, gw.splits, a.D, n, &s.head->count};
        hipLaunchKernelGGL((join_rows_kernel<T>), dim3((unsigned)(up((int64_t)n * a.D / 4, kThreads) / kThreads)), dim3(kThreads), 0, stream, j);
        e = launched();
      }
      return e;
    });
    if (rc != 0) return rc;
  }
  for (int i = 0; i < p.pieces && es == 4; ++i) {
    const int v0 = i * p.columns, n = std::min(p.columns, a.V - v0);
    const float* w = static_cast<const float*>(a.w) + v0 * a.ld_w;
    float* const more = reinterpret_cast<float*>(b.products);
    rc = launch_gemm(product32(b.xc, p.Dp, w, a.ld_w, b.d, p.ldc, a.R, n, a.D, true), true, true, 0, nullptr, stream);
    if (rc != 0) return rc;
    const Rows32 r = {reinterpret_cast<float*>(b.d), p.ldc, p.Rp, n, v0, &s.head->count, b.tc, nullptr, nullptr, s.lse, b.factor};
    hipLaunchKernelGGL(row_grad32_kernel, dim3((a.R + kWaves - 1) / kWaves), dim3(kThreads), 0, stream, r, a.R);
    if (launched() != 0) return -3;
    if (dx != nullptr) {
      float* const out = b.row_parts + (i > 0 ? (int64_t)a.R * a.D : 0);
      rc = launch_gemm(product32(b.d, p.ldc, w, a.ld_w, out, a.D, a.R, a.D, n), true, false, 0, more, stream);
      if (rc == 0 && i > 0) rc = launch_part_sum(b.row_parts, 2, (int64_t)a.R * a.D, b.row_parts, 0, stream);
      if (rc != 0) return rc;
    }
    if (dw != nullptr) {
      rc = launch_gemm(product32(b.d, p.ldc, b.xc, p.Dp, static_cast<float*>(dw) + (int64_t)v0 * a.D, a.D, n, a.D, a.R), false, false, 0, more, stream);
      if (rc != 0) return rc;
    }
  }
  if (dx == nullptr) return 0;
  const JoinArgs j = {b.row_parts, s.rank, b.shift, dx, es == 2 ? ranges((int)up(std::min(a.V, p.columns), kWideK) / kWideK, p.row_splits) : 1, a.D, a.R, nullptr};
  return by_tensor_type(dtype, [&](auto t) {
    hipLaunchKernelGGL((join_rows_kernel<decltype(t)>), dim3((unsigned)(up((int64_t)a.R * a.D / 4, kThreads) / kThreads)), dim3(kThreads), 0, stream, j);
    return launched();
  });
}

}  // namespace castle
