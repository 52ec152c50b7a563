// Mean, sum or each of the cross entropies of hidden rows x [R][D] against a vocabulary w [V][D], without the R x V logits z = x w^T in memory:
//
//   loss r = lse r - z[r][target r],  lse r = log sum_v exp z[r][v]              d[r][v] = g r (exp(z[r][v] - lse r) - [v = target r])
//   dx[r] = sum_v d[r][v] w[v]                                                  dw[v] = sum_r d[r][v] x[r]
//
// Forward: tiles of the product x w^T stay in registers, where each wave reduces its 32 ... 128 columns of a row to a maximum and a sum; these are joined by row.
// Backward: the same product again, turned into d on its way to memory in the 16-bit type, for as many columns of the vocabulary at a time as kPieceBytes hold; two products read a
// piece.  Four products in all, where keeping the logits takes three: what it saves is memory, 2 bytes times R V, and the passes over it.
// What bounds a large call is the matrix units and the card's power: 8192 rows of 2048 over 131072 bf16, 4.4 TFLOP a product, 3.7 ms for the maxima and sums, 4.0 for d, 3.7 for
// either gradient, 1.1 to 1.2 PFLOP/s (the library's product of these sizes 1.36).  Where the contraction is short the ends of the tiles show, which nothing hides behind
// with one workgroup to a CU: 16384 rows of 512 over 32000, 0.54 TFLOP a product, 0.63, 0.73 (1 GB of d written), 0.51 and 0.49 ms.  (Two workgroups of four waves with shorter steps: the same.)
//
// Rows that do not count (target = ignore) are left out at the start: the others are copied together (for both passes), and what the products cost goes with their number, which the kernels
// read from device memory.  So whatever a row that does not count holds, infinities and NaNs too, goes nowhere.
//
// fp32: an element is the sum of three bf16 numbers, 8 bits in each, of any exponent (below 2^-110 it keeps what lies above 2^-134); of the products of two elements' parts the six
// are formed that are not below 2^-24 of the whole.  Operands lie as such parts, 16 first ones, the 16 second ones and the 16 third ones, so a step is 16 of the contraction, and
// everything else is that of the 16-bit types.  (Pairs of fp16 numbers with a power of two for each tensor, three products, took 845 us for 2048 rows of 512 over 32000 instead of 1410, but
// what is far below the largest element loses its digits: the gradient of a class whose softmax values are 2^-40 was gone.  The fp32 products of castle_gemm32.hip convert
// inside the product: logits in memory, 1832 us.)
#include "castle_tiles.h"
#include "castle_dispatch.h"
#include "castle_vocab.h"
#include "castle_wide.h"
#include <algorithm>

namespace castle {
namespace {

constexpr int64_t kPieceBytes = (int64_t)1 << 30;
constexpr int kWaves = kThreads / 64;
constexpr int kCountRows = 1024;   // rows of a workgroup that counts
constexpr int kGatherRows = 16;    // rows of a workgroup that copies
constexpr int kFewLossRows = 4, kLossRows = 16, kManyLossRows = 64;   // rows of a workgroup that joins maxima and sums: of up to 512, of up to 4096 and of more (one atomic of each: 1024 of them 22 us)

// Where maxima start: a score of -inf has weight 0 behind it wherever it stands, and log2(e) times it is finite.
constexpr float kLeast = -0.5f * __FLT_MAX__;

__host__ __device__ constexpr int64_t up(int64_t n, int64_t to) { return (n + to - 1) / to * to; }

// Factors of the rows of d.  d lies in the 16-bit type, so the largest factor is 2^14 ... 2^15, which the gradients lose again (Gain): softmax
// values down to 2^-29 are then normal numbers of fp16 (without it, a mean over 16384 rows would leave nothing of any below 2^-1), and d stays below 2^15.  Where all rows have one
// factor it is 2^15 itself, and the factor goes to the gradients in 32 bits: most rows have -1 or nearly that at their target, and times a factor that
// is no power of two all of these would be rounded the same way, 2^-9 of bf16 at worst.
struct Gain {
  int shift;    // of d, to be taken back
  float gain;   // of the gradients
};
constexpr int kDShift = 15;
// fp32: d is of any size, and the factors are those of the loss, unless the largest is below 2^-20, where the last parts of what is far below it would be lost.
__device__ __forceinline__ int small_factor_shift(float most) { return most > 0.f && most < 0x1p-20f ? -__builtin_amdgcn_frexp_expf(most) : 0; }

// ---- rows that count -----------------------------------------------------------------------------------------------
struct RowArgs {
  VocabArgs v;
  int* block_counts;   // [R / kCountRows], or nullptr: every workgroup counts for itself
  VocabHead* head;
  int32_t* rank;
  void* xc;            // [Rp][Dp]: rows that count, then zero rows up to a multiple of 64 of them; fp32: parts, see split_rows_kernel
  int32_t* tc;         // [Rp] their targets, -1 outside of the vocabulary
  float* tl;           // [Rp] logits of the targets: NaN until they are found
  int32_t* row_of;     // [Rp] the row
  int Dp;
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
// ranks, targets and (16 bits) rows in their order
template <typename T> __global__ __launch_bounds__(kThreads) void gather_rows_kernel(RowArgs a) {
  constexpr int V = elem_traits<T>::vec16;
  typedef vec<T, V> vt;
  __shared__ int s[kWaves], s_rank[kGatherRows];
  const int64_t first = (int64_t)blockIdx.x * kGatherRows;
  int before = 0, total = 0;
  if (a.block_counts != nullptr) {
    const int blocks = (a.v.R + kCountRows - 1) / kCountRows, mine = (int)(first / kCountRows);
    for (int b = threadIdx.x; b < blocks; b += kThreads) {
      const int n = a.block_counts[b];
      total += n;
      before += b < mine ? n : 0;
    }
    for (int64_t r = (int64_t)mine * kCountRows + threadIdx.x; r < first; r += kThreads) before += class_of(a.v, r) != a.v.ignore;
  } else {
#pragma unroll 4
    for (int r = threadIdx.x; r < a.v.R; r += kThreads) {
      const int n = class_of(a.v, r) != a.v.ignore;
      total += n;
      before += r < first ? n : 0;
    }
  }
  before = sum_over_threads<kWaves>(before, s);
  const int all = sum_over_threads<kWaves>(total, s);
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
      a.row_of[rank] = (int32_t)r;
    }
    if (a.v.reduction == kEachLoss && there && !counts) static_cast<T*>(a.loss)[r] = (T)0.f;
  }
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    a.head->count = all;
    a.head->inv_count = 1.f / (float)all;
    a.head->arrived = 0;
  }
  __syncthreads();
  const int pieces = a.Dp / V, have = a.v.D / V;
  if constexpr (sizeof(T) == 2) {   // (fp32: as parts, by a launch of its own)
    const vt none = {};
    for (int k = wave_id(); k < kGatherRows; k += kWaves) {
      const int rank = s_rank[k];
      if (rank >= 0) {
        const T* from = static_cast<const T*>(a.v.x) + (first + k) * a.v.ld_x;
        T* to = static_cast<T*>(a.xc) + (int64_t)rank * a.Dp;
#pragma unroll 4
        for (int i = lane_id(); i < pieces; i += 64) *reinterpret_cast<vt*>(to + i * V) = i < have ? *reinterpret_cast<const vt*>(from + i * V) : none;
      }
      const int64_t r = first + k;   // (the workgroups reach to the next multiple of 64)
      if (r >= all && r < up(all, 64)) {
        T* to = static_cast<T*>(a.xc) + r * a.Dp;
        for (int i = lane_id(); i < pieces; i += 64) *reinterpret_cast<vt*>(to + i * V) = none;
      }
    }
  }
}

// fp32: rows as parts, of 16 columns the first ones, the second and the third ones
struct SplitArgs {
  const float* from;       // rows of ld
  int64_t ld;
  int rows, D, Dp;
  const int32_t* rank;     // nullptr, or where a row goes (-1: nowhere) and `count`, behind which rows up to a multiple of 64 are zero
  const int* count;
  bf16_t* to;              // [rows][3 Dp]
};
constexpr int kPart = 16;   // columns
template <int N> struct Parts { vec<bf16_t, N> p[3]; };
// ANY: a finite number that bf16 rounds to infinity has its largest one as first part
template <bool ANY, int N> __device__ __forceinline__ Parts<N> split_in_three(vec<float, N> x) {
  constexpr float kMost = 0x1.fep127f;
  Parts<N> r;
  vec<float, N> first = x;
  if constexpr (ANY)
#pragma unroll
    for (int e = 0; e < N; ++e) first[e] = fabsf(x[e]) > kMost && fabsf(x[e]) <= __FLT_MAX__ ? copysignf(kMost, x[e]) : x[e];
  r.p[0] = __builtin_convertvector(first, vec<bf16_t, N>);
#pragma unroll
  for (int k = 1; k < 3; ++k) {
    x -= __builtin_convertvector(r.p[k - 1], vec<float, N>);
    r.p[k] = __builtin_convertvector(x, vec<bf16_t, N>);
  }
  return r;
}
// x in the first x_groups workgroups, w in the others
__global__ __launch_bounds__(kThreads) void split_rows_kernel(SplitArgs x_args, SplitArgs w_args, int64_t x_groups) {
  const int64_t group = block_of_many();
  const bool of_x = group < x_groups;
  const SplitArgs& a = of_x ? x_args : w_args;
  const int per = a.Dp / 8;
  const int64_t i = (group - (of_x ? 0 : x_groups)) * kThreads + threadIdx.x, r = i / per;
  if (r >= (a.rank != nullptr ? up(a.rows, 64) : a.rows)) return;
  const int c = (int)(i - r * per) * 8;
  auto put = [&](int64_t row, vec<float, 8> x) __attribute__((always_inline)) {
    const Parts<8> parts = split_in_three<true>(x);
    bf16_t* to = a.to + row * 3 * a.Dp + c / kPart * (3 * kPart) + c % kPart;
#pragma unroll
    for (int k = 0; k < 3; ++k) *reinterpret_cast<frag_mem<bf16_t>*>(to + k * kPart) = parts.p[k];
  };
  vec<float, 8> x = {};
  if (a.rank != nullptr && r >= *a.count && r < up(*a.count, 64)) put(r, x);
  const int64_t row = a.rank == nullptr ? r : r < a.rows ? a.rank[r] : -1;
  if (row < 0) return;
  if (c < a.D) x = *reinterpret_cast<const frag_mem<float>*>(a.from + r * a.ld + c);
  put(row, x);
}

// Maxima and sums of the P column ranges -> log-sum-exp of a row, its loss.  Sums of the losses of a workgroup's rows; the workgroup that arrives last adds them all, in their
// order (a launch of its own took 3 to 5 us).
struct LossArgs {
  const vec<float, 2>* parts;   // [P][Rp]
  VocabHead* head;
  const int32_t* row_of;
  const float* tl;
  float *lse, *sums;
  void* loss;
  int P, reduction;
  int64_t Rp;
};
template <typename T, int ROWS> __global__ __launch_bounds__(kThreads) void row_loss_kernel(LossArgs a) {
  typedef vec<float, 2> v2;
  constexpr int Q = kThreads / ROWS, AT = 8;   // threads of a row, parts of a thread side by side
  __shared__ float s_m[kWaves][ROWS], s_s[kWaves][ROWS];
  const int c = threadIdx.x % ROWS, q = threadIdx.x / ROWS, row = blockIdx.x * ROWS + c, count = a.head->count;
  float m = kLeast, s = 0.f;
  if (row < count)
    for (int p0 = q; p0 < a.P; p0 += AT * Q) {
      v2 x[AT];
      float mn = m;
#pragma unroll
      for (int k = 0; k < AT; ++k) x[k] = p0 + k * Q < a.P ? a.parts[(p0 + k * Q) * a.Rp + row] : v2{kLeast, 0.f};
#pragma unroll
      for (int k = 0; k < AT; ++k) mn = fmaxf(mn, x[k][0]);
      s *= fast_exp2((m - mn) * kLog2e);
#pragma unroll
      for (int k = 0; k < AT; ++k) s += x[k][1] * fast_exp2((x[k][0] - mn) * kLog2e);
      m = mn;
    }
  auto join = [&](float m2, float s2) __attribute__((always_inline)) {
    const float mn = fmaxf(m, m2);
    s = s * fast_exp2((m - mn) * kLog2e) + s2 * fast_exp2((m2 - mn) * kLog2e);
    m = mn;
  };
#pragma unroll
  for (int o = ROWS; o < 64; o <<= 1) {
    const float m2 = __shfl_xor(m, o), s2 = __shfl_xor(s, o);
    join(m2, s2);
  }
  if (lane_id() < ROWS) {
    s_m[wave_id()][c] = m;
    s_s[wave_id()][c] = s;
  }
  __syncthreads();
  float loss = 0.f;
  if (q == 0 && row < count) {
#pragma unroll
    for (int w = 1; w < kWaves; ++w) join(s_m[w][c], s_s[w][c]);
    const float lse = m + logf(s);
    a.lse[row] = lse;
    loss = lse - a.tl[row];
    if (a.reduction == kEachLoss) static_cast<T*>(a.loss)[a.row_of[row]] = (T)loss;
  }
  if (a.reduction == kEachLoss) return;
  __shared__ int s_last;
  __shared__ float s_sum[kWaves];
  if (threadIdx.x < 64) {
#pragma unroll
    for (int o = 1; o < ROWS; o <<= 1) loss += __shfl_xor(loss, o);
    if (threadIdx.x == 0) {
      __hip_atomic_store(a.sums + blockIdx.x, loss, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // (the sum is where every XCD sees it before the count is; release and acquire would write caches back: 1024 workgroups 28 us)
      s_last = __hip_atomic_fetch_add(&a.head->arrived, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == gridDim.x - 1;
    }
  }
  __syncthreads();
  if (!s_last) return;
  float v = 0.f;
  for (int i = threadIdx.x; i < (int)gridDim.x; i += kThreads) v += __hip_atomic_load(a.sums + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) v += __shfl_xor(v, o);
  if (lane_id() == 0) s_sum[wave_id()] = v;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < kWaves; ++w) v += s_sum[w];
    *static_cast<T*>(a.loss) = (T)(a.reduction == kMeanLoss ? v / (float)count : v);
  }
}

// One factor for all rows: 2^15 and the gain (fp32: the factor itself)
template <typename T> __device__ __forceinline__ float one_factor(const void* dloss, const VocabHead& head, int reduction, Gain& gain) {
  float g = (float)*static_cast<const T*>(dloss);
  if (head.count == 0) g = 0.f;
  else if (reduction == kMeanLoss) g *= head.inv_count;
  if constexpr (sizeof(T) == 4) {
    gain = {small_factor_shift(fabsf(g)), 1.f};
    return ldexpf(g, gain.shift);
  }
  gain = {kDShift, g};
  return ldexpf(1.f, kDShift);
}
// kEachLoss: factors of the rows, the largest finite one at 2^14 ... 2^15 (fp32: see small_factor_shift).  fp16: a factor more than 2^kNear below that has a power of two of its own in
// d, which brings it there too, until the gradients of the rows have read it: below 2^-14 of d a number of fp16 loses digits, and over a vocabulary most softmax values of a row are about 2^-15.
// For the gradient of w, which adds over the rows, d then goes to the common power (lower_rows_kernel): what is lost there is 2^-40 of the largest factor.
// (16384 rows of 512 over 32000, forward and backward: 2360 us, with nine of ten rows to be brought there 2640; without the launch 2380.)
constexpr int kNear = 4;
struct FactorArgs {
  const void* dloss;       // [R]
  const int32_t *rank, *tc;
  float* factor;           // [Rp] by rank
  int32_t* own;            // [Rp] by rank, or nullptr: none has a power of its own
  Gain* gain;
  int R;
};
template <typename T> __global__ __launch_bounds__(1024) void factor_kernel(FactorArgs a) {
  __shared__ float s[16];
  const T* g = static_cast<const T*>(a.dloss);
  float most = 0.f;
  for (int r = threadIdx.x; r < a.R; r += 1024)
    if (a.rank[r] >= 0 && fabsf((float)g[r]) <= __FLT_MAX__) most = fmaxf(most, fabsf((float)g[r]));   // (not NaN or infinite)
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) most = fmaxf(most, __shfl_xor(most, o));
  if (lane_id() == 0) s[wave_id()] = most;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < 16; ++w) most = fmaxf(most, s[w]);
  const int shift = sizeof(T) == 4 ? small_factor_shift(most) : most > 0.f ? kDShift - __builtin_amdgcn_frexp_expf(most) : 0;
  if (threadIdx.x == 0 && blockIdx.x == 0) *a.gain = {shift, 1.f};
  for (int64_t r = (int64_t)blockIdx.x * 1024 + threadIdx.x; r < a.R; r += (int64_t)gridDim.x * 1024) {
    const int rank = a.rank[r];
    if (rank < 0) continue;
    float f = a.tc[rank] >= 0 ? ldexpf((float)g[r], shift) : NAN;
    if (a.own != nullptr) {
      const int below = fabsf(f) > 0.f && fabsf(f) <= __FLT_MAX__ ? kDShift - __builtin_amdgcn_frexp_expf(f) : 0, own = below > kNear ? below : 0;
      a.own[rank] = own;
      f = ldexpf(f, own);
    }
    a.factor[rank] = f;
  }
}

// steps of each range of a contraction that is split, the last one may have fewer
__host__ __device__ constexpr int steps_of_range(int steps, int splits) { return steps > 0 ? (steps + splits - 1) / splits : 1; }
__host__ __device__ constexpr int ranges(int steps, int splits) { return (steps + steps_of_range(steps, splits) - 1) / steps_of_range(steps, splits); }

// dx[r] (or dw[v]) = gain 2^-shift times the sum of its partial results, zeros where it does not count
struct JoinArgs {
  const float* parts;   // [splits][R][D]
  const int32_t* rank;
  const Gain* gain;
  const int32_t* own;   // nullptr, or by rank (FactorArgs)
  void* out;
  int splits, D;
  int64_t R;
  const int* count;     // nullptr, or the contraction: there are as many partial results as it has ranges
  int step;             // of the contraction
};
template <typename T> __global__ __launch_bounds__(kThreads) void join_rows_kernel(JoinArgs a) {
  typedef vec<float, 4> v4;
  const int64_t i = block_of_many() * kThreads + threadIdx.x;
  const int per = a.D / 4;
  if (i >= a.R * per) return;
  const int64_t r = i / per;
  const int c = (int)(i - r * per) * 4, rank = a.rank == nullptr ? (int)r : a.rank[r];
  v4 v = {0.f, 0.f, 0.f, 0.f};
  if (rank >= 0) {
    const int splits = a.count != nullptr ? ranges((*a.count + a.step - 1) / a.step, a.splits) : a.splits;
    const float* p = a.parts + (int64_t)rank * a.D + c;
#pragma unroll 4
    for (int k = 0; k < splits; ++k) v += *reinterpret_cast<const v4*>(p + k * a.R * a.D);
    const int shift = a.gain->shift + (a.own != nullptr ? a.own[rank] : 0);
    const float gain = a.gain->gain;
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = ldexpf(v[e], -shift) * gain;
  }
  *reinterpret_cast<vec4_mem<T>*>(static_cast<T*>(a.out) + r * a.D + c) = __builtin_convertvector(v, vec<T, 4>);
}

// The gradients of up to kFewRows rows of 16 bits, where d's rounding at the targets shows: -(1 - p) of a row is its largest element, often by far, and what is lost of it is lost of dx[r] and
// of dw[target] alike (over many rows these errors are as one of the result's own roundings; of four rows of 200 over 904 they were 2.3 times that).  A workgroup to a row, and to 1024
// columns of it: that element again in 32 bits; dx from its partial results and what d has lost there; the row of dw that belongs to the first row of each target once more, all of it,
// with these elements.  (Bound by the trips to memory one behind the other: 64 rows of 512 over 32000, forward and backward in a captured graph, 71 us, with the plain join 66.)
constexpr int kFewRows = 64;
struct FewArgs {
  VocabArgs v;
  const VocabHead* head;
  const int32_t *rank, *tc;
  const float *lse, *factor;   // factor, own: by rank, or nullptr
  const int32_t* own;
  const Gain* gain;
  const void *xc, *d;          // d: one row of blocks
  const float* parts;          // of dx, [splits][R][D]
  void *dx, *dw;
  int Dp, splits;
};
template <typename T> __global__ __launch_bounds__(kThreads) void few_rows_kernel(FewArgs a) {
  constexpr int B = 64;   // rows and columns of a block of d
  typedef vec<float, 4> v4;
  __shared__ float s_sum[kWaves], s_coef[kFewRows];
  const int rank = a.rank[blockIdx.x], lane = lane_id(), wave = wave_id(), D = a.v.D, c = 4 * (blockIdx.y * kThreads + threadIdx.x);
  T* const dx = a.dx != nullptr ? static_cast<T*>(a.dx) + (int64_t)blockIdx.x * D + c : nullptr;
  if (rank < 0) {
    if (dx != nullptr && c < D) st4<T>(dx, vec<T, 4>{});
    return;
  }
  const int target = a.tc[rank], count = min(a.head->count, kFewRows), shift = a.gain->shift;
  const float gain = a.gain->gain;
  const T *x = static_cast<const T*>(a.xc), *w = static_cast<const T*>(a.v.w) + (int64_t)max(target, 0) * a.v.ld_w;
  const T* const d = static_cast<const T*>(a.d) + (int64_t)max(target, 0) / B * (B * B) + max(target, 0) % B;   // of this class, rows B apart
  auto own_of = [&](int k) { return a.own != nullptr ? a.own[k] : 0; };
  // d of row k, whose target this is, by all threads
  auto at_target = [&](int k) {
    float z = 0.f;
    for (int i = 8 * threadIdx.x; i < D; i += 8 * kThreads) {
      const frag<T> p = *reinterpret_cast<const frag_mem<T>*>(x + (int64_t)k * a.Dp + i), q = *reinterpret_cast<const frag_mem<T>*>(w + i);
#pragma unroll
      for (int e = 0; e < 8; ++e) z = __builtin_fmaf((float)p[e], (float)q[e], z);
    }
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) z += __shfl_xor(z, o);
    __syncthreads();   // (the sums before have been read)
    if (lane == 0) s_sum[wave] = z;
    __syncthreads();
    z = 0.f;
#pragma unroll
    for (int i = 0; i < kWaves; ++i) z += s_sum[i];
    return (a.factor != nullptr ? a.factor[k] : ldexpf(1.f, kDShift)) * (fast_exp2((z - a.lse[k]) * kLog2e) - 1.f);
  };
  const int own = own_of(rank);
  float here = 0.f, lost = 0.f;
  if (target >= 0) {
    here = at_target(rank);
    lost = here - (own != 0 ? (float)(T)here : (float)d[rank * B]);   // (a row with a power of its own may have been lowered)
  }
  if (dx != nullptr && c < D) {
    v4 v = {0.f, 0.f, 0.f, 0.f};
    const float* p = a.parts + (int64_t)rank * D + c;
#pragma unroll 4
    for (int k = 0; k < a.splits; ++k) v += *reinterpret_cast<const v4*>(p + (int64_t)k * a.v.R * D);
    const vec<T, 4> there = *reinterpret_cast<const vec4_mem<T>*>(w + c);
    vec<T, 4> out;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float sum = lost != 0.f ? __builtin_fmaf(lost, (float)there[e], v[e]) : v[e];
      out[e] = (T)(ldexpf(sum, -shift - own) * gain);
    }
    st4<T>(dx, out);
  }
  if (a.dw == nullptr || target < 0) return;
  uint64_t same = __ballot(lane < count && a.tc[lane] == target);
  if (same & ((1ull << rank) - 1)) return;   // (another row's)
  if ((int)threadIdx.x < count) s_coef[threadIdx.x] = (float)d[threadIdx.x * B];
  __syncthreads();
  for (; same != 0; same &= same - 1) {
    const int k = __builtin_ctzll(same);
    const float f = ldexpf(k == rank ? here : at_target(k), -own_of(k));
    if (threadIdx.x == 0) s_coef[k] = f;
  }
  __syncthreads();
  if (c >= D) return;
  v4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 8
  for (int k = 0; k < count; ++k) v += s_coef[k] * __builtin_convertvector(*reinterpret_cast<const vec4_mem<T>*>(x + (int64_t)k * a.Dp + c), v4);
#pragma unroll
  for (int e = 0; e < 4; ++e) v[e] = ldexpf(v[e], -shift) * gain;
  st4<T>(static_cast<T*>(a.dw) + (int64_t)target * D + c, __builtin_convertvector(v, vec<T, 4>));
}

// ---- products of 16-bit operands ------------------------------------------------------------------------------------
// The frame is that of gemm_wide_kernel (castle_gemm.hip): tiles of the output by workgroups of eight waves, steps of 64 of the contraction straight from memory to LDS into
// two or three buffers, requested over the end of a tile.  What differs: sizes that are read from device memory, contractions of any length (d and the copied rows are padded with
// zeros, behind the end of a row of w zeros are read, and behind the last row that one again), and what becomes of a tile:
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
  const float *lse, *factor;   // factor: nullptr, or of each row; else one of dloss
  const void* dloss;
  const VocabHead* head;
  int reduction;
  void* c;
  int64_t ldc;
  // kRowGrad: partial results [splits][part_rows][N], added to those that are there; kWeightGrad: c, or partial results [splits][M][N] where there are several
  float* out;
  int64_t part_rows;
  int add;
  Gain* gain;              // kGrad writes it where there is one factor
};

// Loads of a wave for a step.  Of operands that are not contraction-contiguous, parts leave out the quarter that is not used, where that is whole loads: three buffers fit
// the products for dw (2048 rows of 512 over 32000 413 -> 395 us).
template <bool KC, int FREE, bool PARTS> constexpr int kOperandLoads = PARTS && !KC && FREE == 256 ? 3 : FREE / 64;
// PARTS: a step is 16 of the contraction, its first parts at s = 0 of what is in LDS, the second and third ones at 1 and 2; the last quarter of the place is not used (there the
// third ones lie again)
template <typename T, bool KC, int FREE> struct PartsOperand : WideOperand<T, KC, FREE> {
  typedef WideOperand<T, KC, FREE> W;
  static constexpr int N = kOperandLoads<KC, FREE, true>;
  __device__ __forceinline__ void start(const T* p, int64_t ld, int free0, int free_end, int k0) {
    W::at = KC ? p + free0 * ld + 3 * k0 : p + k0 * ld + 3 * free0;
    W::left = free_end - free0;
    place((int)ld, kPart);
  }
  // steps: what is left of the contraction, behind whose end (rows, not contraction-contiguous) the last one is read again
  __device__ __forceinline__ void place(int ld, int steps) {
    const int lane = lane_id(), first = wave_id() * N;
#pragma unroll
    for (int q = 0; q < N; ++q) {
      if constexpr (KC) {
        const int row = 8 * (first + q) + (lane >> 3), piece = (lane & 7) ^ (row >> 1 & 7);
        W::off[q] = 2 * (uint32_t)(ld * min(row, W::left - 1) + 8 * min(piece, 5));
      } else {
        constexpr int PIECES = FREE / 8, ROWS = 64 / PIECES;
        const int k = ROWS * (first + q) + lane / PIECES, p = lane % PIECES ^ 4 * (k & 3), piece = 8 * p < W::left ? p : 0;
        W::off[q] = 2 * (uint32_t)(min(k % kPart, steps - 1) * ld + piece / 2 * (3 * kPart) + min(k / kPart, 2) * kPart + 8 * (piece % 2));
      }
    }
  }
  __device__ __forceinline__ void load(int64_t ld, uint32_t lds) {
#pragma unroll
    for (int q = 0; q < N; ++q) load_to_lds(W::at, W::off[q], lds + 1024 * (wave_id() * N + q));
    W::at += KC ? 3 * kPart : kPart * ld;
  }
};

// d lies in blocks of 64 x 64 (parts: 16 x 16), whole rows of blocks one behind the other, so a step of either product that reads it fetches pieces of 8 KB (parts: 1.5, or whole rows
// of blocks).  (As rows of V, 128 bytes here and there, 64 KB and more apart: the same time where the caches hold a band of columns.)
template <bool PARTS> constexpr int kBlock = PARTS ? kPart : 64;          // rows and columns
template <bool PARTS> constexpr int kBlockRow = PARTS ? 3 * kPart : 64;   // numbers of a row
// Rows of d from a power of two of their own to the common one; workgroups to each row of blocks, most of which have none to do.
struct LowerArgs {
  fp16_t* d;   // [row of blocks][ldc / 64][64][64]
  const int32_t* own;
  const int* count;
  int64_t ldc;
};
__global__ __launch_bounds__(kThreads) void lower_rows_kernel(LowerArgs a) {
  constexpr int B = kBlock<false>, PIECES = B * B / 8, EACH = PIECES / kThreads;   // of a thread, the same rows in every block
  const int64_t first = (int64_t)blockIdx.x * B;
  const int count = *a.count, blocks = (int)(a.ldc / B);
  int own[EACH];
#pragma unroll
  for (int k = 0; k < EACH; ++k) {
    const int64_t r = first + (k * kThreads + threadIdx.x) / (B / 8);
    own[k] = r < count ? a.own[r] : 0;
  }
  for (int b = blockIdx.y; b < blocks; b += gridDim.y)
#pragma unroll
    for (int k = 0; k < EACH; ++k) {
      if (own[k] == 0) continue;
      frag_mem<fp16_t>* p = reinterpret_cast<frag_mem<fp16_t>*>(a.d + first * a.ldc + (int64_t)b * (B * B) + 8 * (k * kThreads + threadIdx.x));
      vec<float, 8> v = __builtin_convertvector((frag<fp16_t>)*p, vec<float, 8>);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = ldexpf(v[e], -own[k]);
      *p = __builtin_convertvector(v, frag<fp16_t>);
    }
}

template <typename T, bool KC, int FREE, bool PARTS> struct BlockOperand : WideOperand<T, KC, FREE> {
  typedef WideOperand<T, KC, FREE> W;
  static constexpr int N = kOperandLoads<KC, FREE, PARTS>, B = kBlock<PARTS>, BR = kBlockRow<PARTS>;
  // p: [row of blocks][ldc / B][B][BR]
  __device__ __forceinline__ void start(const T* p, int64_t ldc, int free0, int free_end, int k0) {
    const int lane = lane_id(), first = wave_id() * N, row_of_blocks = BR * (int)ldc;
    W::left = free_end - free0;
    W::at = p + (KC ? free0 : k0) / B * (int64_t)row_of_blocks + (KC ? k0 : free0) / B * (B * BR);
#pragma unroll
    for (int q = 0; q < N; ++q) {
      if constexpr (KC) {
        const int row = 8 * (first + q) + (lane >> 3), piece = (lane & 7) ^ (row >> 1 & 7), there = min(row, W::left - 1);
        W::off[q] = 2 * (uint32_t)(there / B * row_of_blocks + there % B * BR + 8 * (PARTS ? min(piece, 5) : piece));
      } else {
        constexpr int PIECES = FREE / 8, ROWS = 64 / PIECES, P = B / 8;   // P: pieces of a row of a block, of one part
        const int k = ROWS * (first + q) + lane / PIECES, p = lane % PIECES ^ 4 * (k & 3), piece = 8 * p < W::left ? p : 0;
        W::off[q] = 2 * (uint32_t)(piece / P * (B * BR) + k % B * BR + min(k / B, 2) * B + 8 * (piece % P));
      }
    }
  }
  __device__ __forceinline__ void load(int64_t ldc, uint32_t lds) {
#pragma unroll
    for (int q = 0; q < N; ++q) load_to_lds(W::at, W::off[q], lds + 1024 * (wave_id() * N + q));
    W::at += KC ? (int64_t)B * BR : BR * ldc;
  }
};

// Eight waves over BM x BN: four by two of them for 256 rows, else two by four.
template <int MODE, int BM, int BN, bool PARTS> struct Shape {
  static constexpr int WM = BM == 256 ? 4 : 2, WN = 8 / WM, FM = BM / 32 / WM, FN = BN / 32 / WN;
  static constexpr bool kTurn = MODE == kGrad || (MODE == kWeightGrad && !PARTS);   // a tile goes through LDS to whole rows, 4 KB of each wave
  static constexpr bool kContractA = MODE != kWeightGrad, kContractB = MODE == kStats || MODE == kGrad;   // operands that are contraction-contiguous
  static constexpr int kLoadsA = kOperandLoads<kContractA, BM, PARTS>, kLoads = kLoadsA + kOperandLoads<kContractB, BN, PARTS>;
  static constexpr int kBytesA = kLoadsA * 8 * 1024, kStage = kLoads * 8 * 1024, kTurnBytes = kTurn ? 4096 * 8 : 0;
  static constexpr int kFit = (kMaxLds - kTurnBytes) / kStage, kStages = kFit < 3 ? kFit : 3, kLds = kStages * kStage + kTurnBytes;
  static constexpr int kStores = MODE == kStats ? FM : PARTS && MODE == kGrad ? 6 * FM * FN : MODE == kRowGrad || PARTS ? 4 * FM * FN : 2 * FM * FN;   // of a wave and tile (kWeightGrad: partial results are twice as many)
  static_assert(kStages >= 2 && FM >= 1 && FN >= 1, "");
};
extern __shared__ __attribute__((aligned(16))) unsigned char castle_vocab_lds[];

// END: rows of w end inside a step (kernels of their own: with the test for it in each, 3000 rows of 256 over 50257 took 392 us instead of 383; of 264 636, where reading the row's last piece again took 620)
template <typename T, int MODE, int BM, int BN, bool PARTS, bool END> __global__ __launch_bounds__(kWideThreads, 2) void vocab_product_kernel(ProductArgs a) {
  typedef Shape<MODE, BM, BN, PARTS> S;
  constexpr bool AK = S::kContractA, BKC = S::kContractB;
  constexpr int kStep = PARTS ? kPart : kWideK;   // of the contraction
  typedef std::conditional_t<MODE == kRowGrad || MODE == kWeightGrad, BlockOperand<T, AK, BM, PARTS>, std::conditional_t<PARTS, PartsOperand<T, AK, BM>, WideOperand<T, AK, BM>>> OpA;
  typedef std::conditional_t<PARTS, PartsOperand<T, BKC, BN>, WideOperand<T, BKC, BN>> OpB;
  typedef vec<T, 8> vt;
  const int lane = lane_id(), wave = wave_id(), c = lane & 31, g = lane >> 5;
  const int count = __builtin_amdgcn_readfirstlane(*a.count), M = MODE == kWeightGrad ? a.M : min(a.M, count), K = MODE == kWeightGrad ? (int)up(min(a.K, count), kStep) : a.K;
  const int tiles_m = (M + BM - 1) / BM, tiles_n = (a.N + BN - 1) / BN, tiles = tiles_m * tiles_n;
  float factor = 0.f;
  if constexpr (MODE == kGrad) {
    if (a.factor == nullptr) {
      Gain gain;
      factor = one_factor<std::conditional_t<PARTS, float, T>>(a.dloss, *a.head, a.reduction, gain);
      if (blockIdx.x == 0 && threadIdx.x == 0) *a.gain = gain;
    }
  }
  if (tiles == 0) return;
  // Items are tiles for each range of the contraction; XCD x takes the x-th eighth of them.  Tiles in the order of an XCD's L2: all rows of a band of columns, then those of the next.
  constexpr int kBand = 2048 / BN;
  const int all_steps = (K + kStep - 1) / kStep, per_range = steps_of_range(all_steps, a.splits);
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
    return Item{m * BM, (w.band * kBand + w.rest - m * width) * BN, w.range, w.range * per_range * kStep, min(per_range, all_steps - w.range * per_range)};
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
    // behind the end of the contraction d and the copied rows are zeros, and so are those of parts, to whole steps
    if constexpr (MODE == kRowGrad)
      if (next_k + kStep > K) rb.place((int)a.ldb, K - next_k);
    ra.load(a.lda, lds0 + buffer);
    bool end = false;
    if constexpr (END)
      if ((end = next_k + kStep > K)) rb.load_end(K - next_k, static_cast<const T*>(a.a) + K, lds0 + buffer + S::kBytesA);   // (what is behind the first copied row)
    if (!end) rb.load(a.ldb, lds0 + buffer + S::kBytesA);
    next_k += kStep;
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
  frag<T> fa[PARTS ? 3 : 2][S::FM], fb[2][S::FN];
  auto read_a = [&](int slot, int s) __attribute__((always_inline)) { OpA::read(reinterpret_cast<const T*>(castle_vocab_lds + buffer), fa[slot], wm, s, c, g); };
  auto read_b = [&](int slot, int s) __attribute__((always_inline)) { OpB::read(reinterpret_cast<const T*>(castle_vocab_lds + buffer + S::kBytesA), fb[slot], wn, s, c, g); };
  auto then = []() __attribute__((always_inline)) { __builtin_amdgcn_sched_barrier(0); };   // these reads, then the products of the fragments before
  auto read = [&](int slot, int s) __attribute__((always_inline)) {
    read_a(slot, s);
    read_b(slot, s);
    then();
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
          f[i] = a.factor != nullptr ? a.factor[m] : factor;
        }
      }
    };
    auto rows_are_there = [&]() __attribute__((always_inline)) {
#pragma unroll
      for (int i = 0; i < S::FM; ++i) {
        asm volatile("" : "+v"(t[i]));
        if constexpr (MODE == kGrad) {
          asm volatile("" : "+v"(l[i]), "+v"(f[i]));
          if (t[i] < 0) f[i] = NAN;
        }
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
    auto multiply = [&](int sa, int sb) __attribute__((always_inline)) {
#pragma unroll
      for (int i = 0; i < S::FM; ++i)
#pragma unroll
        for (int j = 0; j < S::FN; ++j) mma(acc[i][j], fb[sb][j], fa[sa][i]);
    };
    for (int it = 0; it < steps; ++it) {
      if constexpr (PARTS) {   // a a', c a', a c', b a', a b', and b b' below
        read_a(1, 2);
        read_b(1, 2);
        then();
        multiply(0, 0);
        read_a(2, 1);
        then();
        multiply(1, 0);
        multiply(0, 1);
        then();
        read_b(1, 1);
        then();
        multiply(2, 0);
        multiply(0, 1);
      } else {
#pragma unroll
        for (int s = 0; s < kWideK / 16 - 1; ++s) {
          read(1 - s % 2, s + 1);
          multiply(s % 2, s % 2);
        }
      }
      arrive();
      done = buffer;
      buffer = buffer == (S::kStages - 1) * S::kStage ? 0 : buffer + S::kStage;
      if (it + 1 < steps) request(done);
      read(0, 0);   // (behind the last step: for nothing)
      multiply(PARTS ? 2 : 1, 1);
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
#pragma unroll
        for (int j = 0; j < S::FN; ++j) {   // (32 columns at a time: of few waves one has a target there, and all wait for it)
          if (__ballot(mine && t[i] / 32 == j) == 0) continue;
          float zt = 0.f;
#pragma unroll
          for (int r = 0; r < 16; ++r) zt = t[i] == 32 * j + acc_row(r, 0) ? z[j][r] : zt;
          if (mine && t[i] / 32 == j) a.tl[m] = zt;
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
    } else if (MODE == kWeightGrad && (PARTS || a.splits > 1)) {   // (of parts, the result itself where the contraction is whole)
      float* out = a.out + (int64_t)range * a.M * a.N;
      const bool result = PARTS && a.splits == 1;
      const int shift = result ? __builtin_amdgcn_readfirstlane(a.gain->shift) : 0;
      const float gain = result ? a.gain->gain : 1.f;
#pragma unroll
      for (int i = 0; i < S::FM; ++i) {
        const int m = m0 + wm + 32 * i + c;
        float* row = out + (int64_t)m * a.N + n0 + wn + 4 * g;
#pragma unroll
        for (int j = 0; j < S::FN; ++j)
#pragma unroll
          for (int q = 0; q < 4; ++q)
            if (m < M && n0 + wn + 32 * j + 8 * q + 4 * g < a.N) {
              vec<float, 4> v = pack4<float>(acc[i][j], q);
              if constexpr (PARTS) {
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = ldexpf(v[e], -shift) * gain;
              }
              *reinterpret_cast<vec<float, 4>*>(row + 32 * j + 8 * q) = v;
            }
        __builtin_amdgcn_sched_barrier(0);
      }
      stored = inside;
    } else {
      // to whole rows through LDS, 32 rows of 64 columns (parts: of 16) at a time, each wave in a place of its own; pieces placed as in the operands
      T* turn = reinterpret_cast<T*>(castle_vocab_lds + S::kStages * S::kStage + wave * 4096);
      const int shift = MODE == kWeightGrad ? __builtin_amdgcn_readfirstlane(a.gain->shift) : 0;
      const float gain = MODE == kWeightGrad ? a.gain->gain : 0.f;
      const int row_end = MODE == kGrad ? min((int)up(count, 64), (int)a.Rp) : M;
#pragma unroll
      for (int i = 0; i < S::FM; ++i) {
        acc_t z[S::FN];
#pragma unroll
        for (int j = 0; j < S::FN; ++j) z[j] = acc[i][j];
        if constexpr (MODE == kGrad) {
          const float shift = l[i] * kLog2e;
          t[i] -= a.first + n0 + wn + 4 * g;
          if (!inside || __ballot(f[i] < 0.f) != 0) {
            const int end = m0 + wm + 32 * i + c < M ? a.N - n0 - wn - 4 * g : 0;
            if (end == 0) t[i] = -1;
#pragma unroll
            for (int j = 0; j < S::FN; ++j)
#pragma unroll
              for (int r = 0; r < 16; ++r) z[j][r] = 32 * j + acc_row(r, 0) < end ? f[i] * fast_exp2(__builtin_fmaf(z[j][r], kLog2e, -shift)) : 0.f;
          } else {   // a factor that is not negative goes to the exponent
            const float up = __builtin_amdgcn_logf(f[i]) - shift;
#pragma unroll
            for (int j = 0; j < S::FN; ++j)
#pragma unroll
              for (int r = 0; r < 16; ++r) z[j][r] = fast_exp2(__builtin_fmaf(z[j][r], kLog2e, up));
          }
#pragma unroll
          for (int j = 0; j < S::FN; ++j) {
            if (__ballot(t[i] >= 0 && t[i] / 32 == j) == 0) continue;
#pragma unroll
            for (int r = 0; r < 16; ++r) z[j][r] -= t[i] == 32 * j + acc_row(r, 0) ? f[i] : 0.f;
          }
        } else {
#pragma unroll
          for (int j = 0; j < S::FN; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) z[j][r] = ldexpf(z[j][r], -shift) * gain;
        }
#pragma unroll
        for (int h = 0; h < (PARTS ? 2 * S::FN : S::FN / 2); ++h) {
          auto put = [&](int p, vec<T, 4> v) __attribute__((always_inline)) { st4<T>(turn + c * 64 + 8 * (p ^ (c >> 1 & 7)) + 4 * g, v); };
          __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
          __builtin_amdgcn_wave_barrier();
          if constexpr (PARTS) {
#pragma unroll
            for (int q = 0; q < 2; ++q) {
              const Parts<4> parts = split_in_three<false>(pack4<float>(z[h / 2], 2 * (h % 2) + q));
#pragma unroll
              for (int k = 0; k < 3; ++k) put(2 * k + q, parts.p[k]);
            }
          } else {
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
              for (int q = 0; q < 4; ++q) put(4 * j + q, pack4<T>(z[2 * h + j], q));
          }
          __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
          __builtin_amdgcn_wave_barrier();
          constexpr int PIECES = PARTS ? 6 : 8;   // of a row
#pragma unroll
          for (int k = 0; k < 32 * PIECES / 64; ++k) {
            const int at = 64 * k + lane, row = at / PIECES, piece = at % PIECES, mm = m0 + wm + 32 * i + row, n = n0 + wn + (PARTS ? 16 * h : 64 * h + 8 * piece);
            const vt v = *reinterpret_cast<const vt*>(turn + row * 64 + 8 * (piece ^ (row >> 1 & 7)));
            constexpr int B = kBlock<PARTS>, BR = kBlockRow<PARTS>;
            T* to = static_cast<T*>(a.c) + (MODE == kGrad ? mm / B * BR * a.ldc + n / B * (B * BR) + mm % B * BR + (PARTS ? 8 * piece : n % B) : mm * a.ldc + n);
            if (mm < row_end && n < (MODE == kGrad ? (int)a.ldc : a.N)) *reinterpret_cast<vt*>(to) = v;
          }
        }
      }
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      stored = inside;
    }
  }
}

template <typename T, int MODE, int BM, int BN, bool PARTS, bool END> int launch_product_as(const ProductArgs& a, hipStream_t stream) {
  typedef Shape<MODE, BM, BN, PARTS> S;
  static PerDeviceOnce once;
  bool& configured = once.flag();
  if (!configured) {
    if (hipFuncSetAttribute(reinterpret_cast<const void*>(&vocab_product_kernel<T, MODE, BM, BN, PARTS, END>), hipFuncAttributeMaxDynamicSharedMemorySize, S::kLds) != hipSuccess) return -3;
    configured = true;
  }
  const int64_t items = up(a.M, BM) / BM * (up(a.N, BN) / BN) * a.splits;
  hipLaunchKernelGGL((vocab_product_kernel<T, MODE, BM, BN, PARTS, END>), dim3((unsigned)std::min<int64_t>(up(items, 8), 256)), dim3(kWideThreads), S::kLds, stream, a);
  return hipGetLastError() == hipSuccess ? 0 : -3;
}
template <typename T, int MODE, int BM, int BN, bool PARTS> int launch_product_t(const ProductArgs& a, hipStream_t stream) {
  if constexpr (!PARTS && (MODE == kStats || MODE == kGrad))
    if (a.K % kWideK != 0) return launch_product_as<T, MODE, BM, BN, PARTS, true>(a, stream);
  return launch_product_as<T, MODE, BM, BN, PARTS, false>(a, stream);
}
// Rows and columns of a workgroup's tile.  Of 64, 128 or 256 rows those with which the fullest CU is done first (us): 1.4 a step and 5 an end of 256 x 256, 0.85 and 3 of 128,
// 0.56 and 1.6 of 64.  (The loss alone of 128 rows over 32000, 512 wide in bf16, with tiles of 64 rows / 128: 28 / 30 us, 2048 wide 46 / 52; 256 rows 34 / 32, since 500 tiles take two rounds.)
struct Tile { int rows, columns; };
int64_t tiles(int64_t m, int64_t n, Tile t) { return up(m, t.rows) / t.rows * (up(n, t.columns) / t.columns); }
Tile tile_of(int R, int n, int steps) {
  auto cost = [&](Tile t, double step, double end) { return (tiles(R, n, t) + 255) / 256 * (step * steps + end); };
  const double large = cost({256, 256}, 1.4, 5), middle = cost({128, 256}, 0.85, 3), small = cost({64, 256}, 0.56, 1.6);
  return R <= 64 || small < std::min(middle, large) ? Tile{64, 256} : middle < large ? Tile{128, 256} : Tile{256, 256};
}
template <int MODE> int launch_product(const ProductArgs& a, Tile tile, int dtype, hipStream_t stream) {
  auto of_type = [&](auto t, auto parts) {
    using T = decltype(t);
    constexpr bool P = decltype(parts)::value;
    if constexpr (MODE != kWeightGrad) {
      if (tile.rows == 64) {
        if constexpr (MODE == kRowGrad)
          if (tile.columns == 128) return launch_product_t<T, MODE, 64, 128, P>(a, stream);
        return launch_product_t<T, MODE, 64, 256, P>(a, stream);
      }
      if (tile.rows == 128) return launch_product_t<T, MODE, 128, 256, P>(a, stream);
    }
    if constexpr (MODE == kRowGrad || MODE == kWeightGrad)
      if (tile.columns == 128) return launch_product_t<T, MODE, 256, 128, P>(a, stream);
    return launch_product_t<T, MODE, 256, 256, P>(a, stream);
  };
  switch (dtype) {
    case 0: return of_type(bf16_t(), std::true_type());
    case 1: return of_type(bf16_t(), std::false_type());
    case 2: return of_type(fp16_t(), std::false_type());
    default: return -1;
  }
}

// ---- sizes ----------------------------------------------------------------------------------------------------------
int loss_rows(int R) { return R > 4096 ? kManyLossRows : R > 512 ? kLossRows : kFewLossRows; }
int loss_groups(int R) { return (R + loss_rows(R) - 1) / loss_rows(R); }
struct Split { Tile tile; int ranges; };   // of a contraction
struct Plan {
  int64_t Rp;              // rows, a multiple of 64
  int Dp;                  // width of a copied row
  int P;                   // column ranges of a row's maxima and sums
  int columns, pieces;     // of the vocabulary at a time
  int64_t ldc;             // of d
  Tile logits;
  Split rows, weights;
  int step;                // of a contraction
};
// Tile and ranges of a contraction of `steps` for m x n outputs, from what it takes roughly (us): so much a step and an end for each of the items of the fullest CU, and for
// several ranges their partial results, written and read at 4 TB/s.  (Forward pass and the gradient of the rows over 32000, 512 wide in bf16, without tiles of 64 rows / with them:
// 64 rows 67 / 61 us, 128 76 / 68, 256 81 / 78; over 4000 256 61 / 56, 1000 69 / 65.)
Split split_of(int64_t m, int64_t n, int64_t steps, std::initializer_list<Tile> kinds) {
  Split best = {};
  double best_cost = 1e30;
  for (const Tile t : kinds) {
    const int area = t.rows * t.columns;
    const double step = area > 128 * 256 ? 1.5 : area > 64 * 256 ? 1.05 : area > 64 * 128 ? 0.8 : 0.6, end = area > 128 * 256 ? 5 : 3;
    const int most = (int)std::min<int64_t>(128, std::max<int64_t>(1, steps / 2));
    const int64_t items = tiles(m, n, t);
    for (int s = 1; s <= most; ++s) {
      const double cost = (items * s + 255) / 256 * (step * steps_of_range((int)steps, s) + end) + (s > 1 ? 8e-6 / 4 * s * m * n : 0);
      if (cost < best_cost) {
        best_cost = cost;
        best = {t, s};
      }
    }
  }
  return best;
}
// bytes of an element of an operand of the products; es: of one of the tensors
constexpr int operand_bytes(int es) { return es == 4 ? 6 : 2; }
Plan make_plan(const VocabArgs& a, int es, bool gradients) {
  Plan p = {};
  p.step = es == 4 ? kPart : kWideK;
  p.Rp = up(a.R, 64);
  p.Dp = (int)up(a.D, p.step);
  const int64_t fit = std::max<int64_t>(256, kPieceBytes / (p.Rp * operand_bytes(es)) / 256 * 256), width = up(a.V, 64);
  p.pieces = (int)((width + fit - 1) / fit);
  p.columns = (int)up((a.V + p.pieces - 1) / p.pieces, 256);
  p.pieces = (a.V + p.columns - 1) / p.columns;
  p.ldc = std::min<int64_t>(p.columns, width);
  p.logits = tile_of(a.R, a.V, p.Dp / p.step);
  p.P = (int)(up(a.V, 256) / 256 * (p.logits.rows == 256 ? 2 : 4));
  if (!gradients) return p;
  const int wide = a.D <= 128 ? 128 : 256;
  p.rows = wide == 128 ? (a.R <= 64 ? split_of(a.R, a.D, p.ldc / p.step, {{64, 128}}) : split_of(a.R, a.D, p.ldc / p.step, {{64, 128}, {256, 128}}))
         : a.R <= 64   ? split_of(a.R, a.D, p.ldc / p.step, {{64, 128}, {64, 256}})
                       : split_of(a.R, a.D, p.ldc / p.step, {{64, 128}, {64, 256}, {128, 256}, {256, 256}});
  p.weights = split_of(p.ldc, a.D, p.Rp / p.step, {{256, wide}});
  return p;
}
// A call asks three times for the plan of its sizes, 2 us each: a thread keeps the last one.
Plan plan(const VocabArgs& a, int es, bool gradients) {
  struct Last { int R, V, D, es, gradients; Plan p; };
  static thread_local Last last = {};
  if (last.R != a.R || last.V != a.V || last.D != a.D || last.es != es || last.gradients != (int)gradients) last = {a.R, a.V, a.D, es, gradients, make_plan(a, es, gradients)};
  return last.p;
}
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
  char *xc, *wc;   // fp32: the parts of the rows that count and of w
  int32_t* row_of;
  float *tl, *sums;
  vec<float, 2>* parts;
  Fwd(const VocabArgs& a, const Plan& p, int es, Carve& c) {
    block_counts = c.take<int>(up(a.R, kCountRows) / kCountRows);
    xc = c.take<char>(es == 4 ? p.Rp * p.Dp * operand_bytes(es) : 0);
    wc = c.take<char>(es == 4 ? (int64_t)a.V * p.Dp * operand_bytes(es) : 0);
    tl = c.take<float>(p.Rp);
    row_of = c.take<int32_t>(p.Rp);
    sums = c.take<float>(loss_groups(a.R));
    parts = c.take<vec<float, 2>>(p.P * p.Rp);
  }
};
struct Bwd {
  char *xc, *wc;
  float* factor;
  int32_t* own;
  Gain* gain;
  char* d;
  float *row_parts, *weight_parts;
  Bwd(const VocabArgs& a, const Plan& p, int es, bool need_x, bool need_w, Carve& c) {
    xc = c.take<char>(es == 4 ? p.Rp * p.Dp * operand_bytes(es) : 0);
    wc = c.take<char>(es == 4 ? (int64_t)a.V * p.Dp * operand_bytes(es) : 0);
    factor = c.take<float>(p.Rp);
    own = c.take<int32_t>(p.Rp);
    gain = c.take<Gain>(1);
    d = c.take<char>(p.Rp * p.ldc * operand_bytes(es));
    row_parts = c.take<float>(need_x ? (int64_t)p.rows.ranges * a.R * a.D : 0);
    weight_parts = c.take<float>(need_w && p.weights.ranges > 1 ? p.weights.ranges * p.ldc * a.D : 0);
  }
};
struct State {
  VocabHead* head;
  int32_t *rank, *tc;
  float* lse;
  char* xc;   // 16 bits: the rows that count
  State(int64_t R, int D, int es, Carve& c) {
    head = c.take<VocabHead>(1);
    rank = c.take<int32_t>(R);
    tc = c.take<int32_t>(R);
    lse = c.take<float>(R);
    xc = c.take<char>(es == 2 ? up(R, 64) * up(D, kWideK) * 2 : 0);
  }
};
int launched() { return hipGetLastError() == hipSuccess ? 0 : -3; }
int launch_gather(const RowArgs& a, int dtype, hipStream_t stream) {
  return by_tensor_type(dtype, [&](auto t) {
    using T = decltype(t);
    hipLaunchKernelGGL((gather_rows_kernel<T>), dim3((unsigned)(up(a.v.R, 64) / kGatherRows)), dim3(kThreads), 0, stream, a);
    return launched();
  });
}

// fp32: the rows of x that count, and w, as parts
int launch_split(const VocabArgs& a, const Plan& p, const int* count, const int32_t* rank, void* xc, void* wc, hipStream_t stream) {
  const SplitArgs x = {static_cast<const float*>(a.x), a.ld_x, a.R, a.D, p.Dp, rank, count, static_cast<bf16_t*>(xc)};
  const SplitArgs w = {static_cast<const float*>(a.w), a.ld_w, a.V, a.D, p.Dp, nullptr, nullptr, static_cast<bf16_t*>(wc)};
  auto groups = [&](int64_t rows) { return up(rows * (p.Dp / 8), kThreads) / kThreads; };
  hipLaunchKernelGGL(split_rows_kernel, many_blocks(groups(p.Rp) + groups(a.V)), dim3(kThreads), 0, stream, x, w, groups(p.Rp));
  return launched();
}

}  // namespace

int64_t vocab_state_bytes(int64_t R, int D, int es) {
  Carve c = {nullptr};
  State(R, D, es, c);
  return c.used;
}
int64_t vocab_fwd_bytes(const VocabArgs& a, int es) {
  Carve c = {nullptr};
  Fwd(a, plan(a, es, false), es, c);
  return c.used;
}
int64_t vocab_bwd_bytes(const VocabArgs& a, int es, bool need_x, bool need_w) {
  Carve c = {nullptr};
  Bwd(a, plan(a, es, true), es, need_x, need_w, c);
  return c.used;
}

int launch_vocab_fwd(const VocabArgs& a, int dtype, void* loss, void* state, void* workspace, hipStream_t stream) {
  const int es = dtype == 0 ? 4 : 2;
  const Plan p = plan(a, es, false);
  Carve cs = {static_cast<char*>(state)}, cw = {static_cast<char*>(workspace)};
  const State s(a.R, a.D, es, cs);
  const Fwd f(a, p, es, cw);
  char* const xc = es == 4 ? f.xc : s.xc;
  const bool count = a.R > 4096;   // (up to there the copying workgroups count for themselves, which is less than a launch)
  const RowArgs rows = {a, count ? f.block_counts : nullptr, s.head, s.rank, xc, s.tc, f.tl, f.row_of, p.Dp, loss};
  if (count) hipLaunchKernelGGL(count_rows_kernel, dim3((unsigned)(up(a.R, kCountRows) / kCountRows)), dim3(kThreads), 0, stream, rows);
  int rc = launch_gather(rows, dtype, stream);
  if (rc == 0 && es == 4) rc = launch_split(a, p, &s.head->count, s.rank, f.xc, f.wc, stream);
  if (rc != 0) return rc;
  ProductArgs g = {};
  g.a = xc;
  g.b = es == 4 ? f.wc : a.w;
  g.lda = es == 4 ? 3 * p.Dp : p.Dp;
  g.ldb = es == 4 ? 3 * p.Dp : a.ld_w;
  g.M = a.R;
  g.N = a.V;
  g.K = a.D;
  g.count = &s.head->count;
  g.splits = 1;
  g.parts = f.parts;
  g.tl = f.tl;
  g.Rp = p.Rp;
  g.tc = s.tc;
  rc = launch_product<kStats>(g, p.logits, dtype, stream);
  if (rc != 0) return rc;
  const LossArgs l = {f.parts, s.head, f.row_of, f.tl, s.lse, f.sums, loss, p.P, a.reduction, p.Rp};
  return by_tensor_type(dtype, [&](auto t) {
    auto go = [&](auto rows) { hipLaunchKernelGGL((row_loss_kernel<decltype(t), rows.value>), dim3(loss_groups(a.R)), dim3(kThreads), 0, stream, l); };
    switch (loss_rows(a.R)) {
      case kFewLossRows: go(std::integral_constant<int, kFewLossRows>()); break;
      case kLossRows: go(std::integral_constant<int, kLossRows>()); break;
      default: go(std::integral_constant<int, kManyLossRows>());
    }
    return launched();
  });
}

int launch_vocab_bwd(const VocabArgs& a, int dtype, const void* dloss, const void* state, void* dx, void* dw, void* workspace, hipStream_t stream) {
  const int es = dtype == 0 ? 4 : 2;
  const Plan p = plan(a, es, true);
  Carve cs = {static_cast<char*>(const_cast<void*>(state))}, cw = {static_cast<char*>(workspace)};
  const State s(a.R, a.D, es, cs);
  const Bwd b(a, p, es, dx != nullptr, dw != nullptr, cw);
  char* const xc = es == 4 ? b.xc : s.xc;
  int rc = es == 4 ? launch_split(a, p, &s.head->count, s.rank, b.xc, b.wc, stream) : 0;
  int32_t* const own = dtype == 2 && a.reduction == kEachLoss ? b.own : nullptr;
  if (rc == 0 && a.reduction == kEachLoss) {
    const FactorArgs f = {dloss, s.rank, s.tc, b.factor, own, b.gain, a.R};
    rc = by_tensor_type(dtype, [&](auto t) {
      hipLaunchKernelGGL((factor_kernel<decltype(t)>), dim3(std::min<unsigned>(64, (unsigned)(up(a.R, 1024) / 1024))), dim3(1024), 0, stream, f);
      return launched();
    });
  }
  auto join = [&](const JoinArgs& j) {
    return by_tensor_type(dtype, [&](auto t) {
      hipLaunchKernelGGL((join_rows_kernel<decltype(t)>), many_blocks(up(j.R * j.D / 4, kThreads) / kThreads), dim3(kThreads), 0, stream, j);
      return launched();
    });
  };
  const int64_t ld_x = es == 4 ? 3 * p.Dp : p.Dp, ld_w = es == 4 ? 3 * p.Dp : a.ld_w;   // numbers of 2 bytes
  for (int i = 0; i < p.pieces && rc == 0; ++i) {
    const int v0 = i * p.columns, n = std::min(p.columns, a.V - v0);
    ProductArgs g = {};
    g.a = xc;
    g.b = (es == 4 ? b.wc : static_cast<const char*>(a.w)) + v0 * ld_w * 2;
    g.lda = ld_x;
    g.ldb = ld_w;
    g.M = a.R;
    g.N = n;
    g.K = a.D;
    g.count = &s.head->count;
    g.splits = 1;
    g.Rp = p.Rp;
    g.tc = s.tc;
    g.first = v0;
    g.lse = s.lse;
    g.factor = a.reduction == kEachLoss ? b.factor : nullptr;
    g.dloss = dloss;
    g.head = s.head;
    g.reduction = a.reduction;
    g.c = b.d;
    g.ldc = p.ldc;
    g.gain = b.gain;
    rc = launch_product<kGrad>(g, p.logits, dtype, stream);
    if (rc == 0 && dx != nullptr) {
      ProductArgs x = g;
      x.a = b.d;
      x.lda = p.ldc;
      x.N = a.D;
      x.K = n;
      x.splits = p.rows.ranges;
      x.out = b.row_parts;
      x.part_rows = a.R;
      x.add = i > 0;
      rc = launch_product<kRowGrad>(x, p.rows.tile, dtype, stream);
    }
    if (rc == 0 && dw != nullptr && own != nullptr) {
      const int64_t rows = p.Rp / kBlock<false>;
      hipLaunchKernelGGL(lower_rows_kernel, dim3((unsigned)rows, (unsigned)std::max<int64_t>(1, std::min(p.ldc / kBlock<false>, 1024 / rows))), dim3(kThreads), 0, stream,
                         LowerArgs{reinterpret_cast<fp16_t*>(b.d), own, &s.head->count, p.ldc});
      rc = launched();
    }
    if (rc == 0 && dw != nullptr) {
      ProductArgs w = g;
      w.a = b.d;
      w.lda = p.ldc;
      w.b = xc;
      w.ldb = ld_x;
      w.M = n;
      w.N = a.D;
      w.K = a.R;
      w.splits = p.weights.ranges;
      w.c = static_cast<char*>(dw) + (int64_t)v0 * a.D * es;
      w.ldc = a.D;
      w.out = w.splits > 1 ? b.weight_parts : static_cast<float*>(w.c);
      rc = launch_product<kWeightGrad>(w, p.weights.tile, dtype, stream);
      if (rc == 0 && w.splits > 1)
        rc = join({b.weight_parts, nullptr, b.gain, nullptr, w.c, w.splits, a.D, n, &s.head->count, p.step});
    }
  }
  if (rc != 0) return rc;
  if (es == 2 && a.R <= kFewRows) {   // (of so few rows d is one piece for any vocabulary, and its contraction for dw is one range)
    const FewArgs f = {a, s.head, s.rank, s.tc, s.lse, a.reduction == kEachLoss ? b.factor : nullptr, own, b.gain, xc, b.d, b.row_parts, dx, dw, p.Dp,
                       ranges((int)up(std::min(a.V, p.columns), p.step) / p.step, p.rows.ranges)};
    const dim3 grid((unsigned)a.R, (unsigned)(up(a.D, 4 * kThreads) / (4 * kThreads)));
    if (dtype == 1) hipLaunchKernelGGL((few_rows_kernel<bf16_t>), grid, dim3(kThreads), 0, stream, f);
    else hipLaunchKernelGGL((few_rows_kernel<fp16_t>), grid, dim3(kThreads), 0, stream, f);
    return launched();
  }
  if (dx == nullptr) return rc;
  return join({b.row_parts, s.rank, b.gain, own, dx, ranges((int)up(std::min(a.V, p.columns), p.step) / p.step, p.rows.ranges), a.D, a.R, nullptr, p.step});
}

}  // namespace castle
