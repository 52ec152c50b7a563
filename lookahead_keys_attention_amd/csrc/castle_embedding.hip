// Token embedding of any vocabulary: rows of the table times a scale, and the table's gradient by sorted tokens.
//
//   y[r] = scale table[token r]          dtable[v] = scale sum over the r whose token is v of dy[r]
//
// Both are bound by HBM: the forward pass reads a row and writes one, the gradient reads dy and writes the whole table once.  The gradient needs the rows of
// each token together, in an order of their own (atomic additions would leave the order, and with it the last bits, to chance): (token, place) pairs are sorted, stable, by
// digits of up to ten bits, a counting and a placing launch for each.  Where each token's places begin and end is noted, and pieces of 64 sorted places that hold one
// token alone are summed first, so that a token that takes a tenth of a text does not keep one workgroup busy when the rest is done; then every row of the
// table is summed and written once, zeros where there is no token.
// Measured, bf16: 65536 tokens over 131072 rows of 2048, forward 86 us (5.5 TB/s), gradient 212 (3.8 TB/s of what it has to move, 33 of it the sort); 16384 over 32000 of 512, 7 and
// 44 us, of which 24 are the four launches of the sort, each little more than its start and two trips to memory.
#include "castle_tiles.h"
#include "castle_dispatch.h"
#include "castle_tokens.h"
#include <algorithm>

namespace castle {
namespace {

constexpr int kWaves = kThreads / 64;
constexpr int kRun = 64;   // sorted places of a piece

__device__ __forceinline__ int64_t token_of(const TokenRows& t, int64_t r) {
  if (t.n == t.rows) return t.index[r];
  const uint32_t q = (uint32_t)r / (uint32_t)t.n;   // (rows are fewer than 2^31)
  return t.index[q * t.index_ld + ((uint32_t)r - q * (uint32_t)t.n)];
}

// N elements at a time: 16 bytes, wherever they begin, or one element where a row has fewer.  Piece i of a row: the last one ends with the row, and reads and writes what the
// one before it does as well (single elements where rows are no whole pieces: 5569 tokens of 828 bf16 over 6556, forward and gradient, 121 us, so 58).
// (Widths and vocabularies reach 2^31 - 1: what is a little more than they are is formed in 32 bits without a sign, or in 64.)
template <int N> __device__ __forceinline__ int column(int i, int D) { return (int)min((uint32_t)i * N, (uint32_t)D - N); }
template <int N> __host__ __device__ __forceinline__ int pieces_of(int D) { return (int)(((uint32_t)D + N - 1) / N); }
template <typename T, int N> struct Anywhere { typedef vec<T, N> type __attribute__((aligned(sizeof(T)))); };
template <typename T, int N> __device__ __forceinline__ vec<float, N> load_n(const T* p) {
  const vec<T, N> v = *reinterpret_cast<const typename Anywhere<T, N>::type*>(p);
  return __builtin_convertvector(v, vec<float, N>);
}
template <typename T, int N> __device__ __forceinline__ void store_n(T* p, vec<float, N> v) { *reinterpret_cast<typename Anywhere<T, N>::type*>(p) = __builtin_convertvector(v, vec<T, N>); }
template <int N> __device__ __forceinline__ vec<float, N> fill_n(float x) {
  vec<float, N> v;
#pragma unroll
  for (int e = 0; e < N; ++e) v[e] = x;
  return v;
}

// LPR lanes to a row
template <typename T, int N, int LPR> __global__ __launch_bounds__(kThreads) void embedding_kernel(EmbeddingArgs a) {
  constexpr int RPG = kThreads / LPR;
  const int64_t r = block_of_many() * RPG + threadIdx.x / LPR;
  if (r >= a.tokens.rows) return;
  const int64_t t = token_of(a.tokens, r);
  const bool there = t >= 0 && t < a.V;
  const T* row = static_cast<const T*>(a.table) + (there ? t : 0) * a.ld;
  T* y = static_cast<T*>(a.y) + r * a.D;
#pragma unroll 4
  for (int i = threadIdx.x % LPR; i < pieces_of<N>(a.D); i += LPR) {
    const int c = column<N>(i, a.D);
    const vec<float, N> v = load_n<T, N>(row + c) * a.scale;
    store_n<T, N>(y + c, there ? v : fill_n<N>(NAN));
  }
}

// ---- sorting -------------------------------------------------------------------------------------------------------
// Every wave has a range of its own, in order; workgroup g has those of four waves.
struct Range { uint32_t first, end; };   // sorted places of a token
struct SortArgs {
  TokenRows tokens;
  int V, padding;
  int shift, bits;
  int64_t wave_tokens;
  const uint32_t *keys_in, *places_in;   // nullptr: the tokens themselves
  uint32_t *keys, *places;
  uint32_t* counts;                      // [workgroup][digit]
  // workgroups behind the `groups` that sort clear ranges of sorted places in passing, where there are any
  Range* ranges;
  int groups;
};
constexpr int kClear = 4096;   // ranges of a workgroup that clears
__device__ __forceinline__ void clear_ranges(const SortArgs& a, int threads) {
  const int64_t first = (int64_t)(blockIdx.x - a.groups) * kClear;
  for (int64_t v = first + threadIdx.x; v < min((int64_t)a.V, first + kClear); v += threads) a.ranges[v] = {0, 0};
}
__device__ __forceinline__ uint32_t key_of(const SortArgs& a, int64_t i) {
  if (a.keys_in != nullptr) return a.keys_in[i];
  const int64_t t = token_of(a.tokens, i);
  return t >= 0 && t < a.V && t != a.padding ? (uint32_t)t : (uint32_t)a.V;   // behind all others
}
extern __shared__ __attribute__((aligned(16))) uint32_t castle_digits[];   // [wave][digit]
// how many of each digit there are in the range of this wave
__device__ __forceinline__ void wave_counts(const SortArgs& a, uint32_t* mine, int64_t first, int64_t last) {
  for (int64_t i = first + lane_id(); i < last; i += 64) atomicAdd(mine + (key_of(a, i) >> a.shift & ((1u << a.bits) - 1)), 1u);
}
__global__ __launch_bounds__(kThreads) void sort_count_kernel(SortArgs a) {
  const int digits = 1 << a.bits;
  if ((int)blockIdx.x >= a.groups) return clear_ranges(a, kThreads);
  for (int d = threadIdx.x; d < digits; d += kThreads) castle_digits[d] = 0;
  __syncthreads();
  const int64_t first = ((int64_t)blockIdx.x * kWaves + wave_id()) * a.wave_tokens;
  wave_counts(a, castle_digits, first, min(a.tokens.rows, first + a.wave_tokens));
  __syncthreads();
  for (int d = threadIdx.x; d < digits; d += kThreads) a.counts[(int64_t)blockIdx.x * digits + d] = castle_digits[d];
}
// From the counts of all workgroups to the place of each digit's first key of each wave here, then the keys to their places: equal digits in the order they came.
__global__ __launch_bounds__(kThreads) void sort_place_kernel(SortArgs a) {
  const int digits = 1 << a.bits, wave = wave_id(), lane = lane_id();
  __shared__ uint32_t s_sum[kWaves];
  for (int d = threadIdx.x; d < kWaves * digits; d += kThreads) castle_digits[d] = 0;
  __syncthreads();
  const int64_t first = ((int64_t)blockIdx.x * kWaves + wave) * a.wave_tokens, last = min(a.tokens.rows, first + a.wave_tokens);
  uint32_t* const mine = castle_digits + wave * digits;
  wave_counts(a, mine, first, last);
  // a thread has `per` digits in a row
  const int per = max(1, digits / kThreads), d0 = threadIdx.x * per;
  constexpr int kMaxPer = 4;
  uint32_t before[kMaxPer] = {}, all[kMaxPer] = {}, sum = 0;
  if (d0 < digits) {
#pragma unroll
    for (int p = 0; p < kMaxPer; ++p) {
      if (p >= per) break;
#pragma unroll 16
      for (int g = 0; g < a.groups; ++g) {
        const uint32_t n = a.counts[(int64_t)g * digits + d0 + p];
        all[p] += n;
        before[p] += g < (int)blockIdx.x ? n : 0;
      }
      sum += all[p];
    }
  }
  uint32_t up = sum;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const uint32_t left = __shfl_up(up, o);
    up += lane >= o ? left : 0;
  }
  if (lane == 63) s_sum[wave] = up;
  __syncthreads();
  if (d0 < digits) {
    uint32_t at = up - sum;
#pragma unroll
    for (int w = 0; w < kWaves - 1; ++w) at += w < wave ? s_sum[w] : 0;
#pragma unroll
    for (int p = 0; p < kMaxPer; ++p) {
      if (p >= per) break;
      uint32_t place = at + before[p];
      at += all[p];
#pragma unroll
      for (int w = 0; w < kWaves; ++w) {
        const uint32_t n = castle_digits[w * digits + d0 + p];
        castle_digits[w * digits + d0 + p] = place;
        place += n;
      }
    }
  }
  __syncthreads();
  for (int64_t base = first; base < last; base += 64) {
    const int64_t i = base + lane;
    const bool there = i < last;
    const uint32_t key = there ? key_of(a, i) : 0, d = key >> a.shift & (digits - 1);
    uint64_t same = __ballot(there);   // lanes of the same digit
    for (int b = 0; b < a.bits; ++b) {
      const uint64_t ones = __ballot(d >> b & 1);
      same &= d >> b & 1 ? ones : ~ones;
    }
    const uint64_t below = (1ull << lane) - 1;
    uint32_t at = 0;
    if (there) at = mine[d] + __popcll(same & below);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    if (there && (same & below) == 0) mine[d] += __popcll(same);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    if (there) {
      a.keys[at] = key;
      a.places[at] = a.places_in != nullptr ? a.places_in[i] : (uint32_t)i;
    }
  }
}

// Up to 8192 tokens and 2^18 keys: all in one workgroup of sixteen waves, a pair in one word, eight of them in the registers of a thread, from there to their places in LDS and
// back.  Lanes of equal digits are found once a pass: a pair's rank among the digits of its wave is kept until the places are known (32000 rows of 512 bf16, the
// whole gradient: 8192 tokens 38 us, 8256 by four launches 45; the 16384 of which four launches sort in 25 us take a workgroup 34).
constexpr int kSortRounds = 8, kSortThreads = 1024, kSortTokens = kSortRounds * kSortThreads, kPlaceBits = 13;
template <int BITS> __global__ __launch_bounds__(kSortThreads) void sort_all_kernel(SortArgs a, int passes) {
  constexpr int W = kSortThreads / 64, DIGITS = 1 << BITS;
  if ((int)blockIdx.x >= a.groups) return clear_ranges(a, kSortThreads);
  const int wave = wave_id(), lane = lane_id(), n = (int)a.tokens.rows;
  uint32_t* const s_pairs = castle_digits;                  // [kSortTokens]
  uint32_t* const s_digits = s_pairs + kSortTokens;         // [wave][digit]
  uint32_t* const mine = s_digits + wave * DIGITS;
  __shared__ uint32_t s_sum[W];
  // of each wave a range in order, 64 at a time
  const int per_wave = ((n + W - 1) / W + 63) / 64 * 64, first = wave * per_wave, last = min(n, first + per_wave);
  uint32_t e[kSortRounds], rank[kSortRounds];
#pragma unroll
  for (int i = 0; i < kSortRounds; ++i) {
    const int at = first + 64 * i + lane;
    e[i] = at < last ? key_of(a, at) << kPlaceBits | (uint32_t)at : 0;
  }
  for (int pass = 0; pass < passes; ++pass) {
    const int shift = kPlaceBits + pass * BITS;
    for (int d = threadIdx.x; d < W * DIGITS; d += kSortThreads) s_digits[d] = 0;
    __syncthreads();
    const uint64_t below = (1ull << lane) - 1;
#pragma unroll
    for (int i = 0; i < kSortRounds; ++i) {
      if (first + 64 * i >= last) break;
      const bool there = first + 64 * i + lane < last;
      const uint32_t d = e[i] >> shift & (DIGITS - 1);
      uint64_t same = __ballot(there);   // lanes of the same digit
#pragma unroll
      for (int b = 0; b < BITS; ++b) {
        const uint64_t ones = __ballot(d >> b & 1);
        same &= d >> b & 1 ? ones : ~ones;
      }
      const uint32_t before = mine[d];
      rank[i] = before + __popcll(same & below);
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
      if (there && (same & below) == 0) mine[d] = before + __popcll(same);
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
    }
    __syncthreads();
    // the place of each digit's first pair of each wave: a thread has one digit (there are at most as many as threads)
    const bool digit = (int)threadIdx.x < DIGITS;
    uint32_t count[W], sum = 0;
#pragma unroll
    for (int w = 0; w < W; ++w) {
      count[w] = digit ? s_digits[w * DIGITS + threadIdx.x] : 0;
      sum += count[w];
    }
    uint32_t up = sum;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const uint32_t left = __shfl_up(up, o);
      up += lane >= o ? left : 0;
    }
    if (lane == 63) s_sum[wave] = up;
    __syncthreads();
    uint32_t at = up - sum;
    for (int w = 0; w < wave; ++w) at += s_sum[w];
    if (digit) {
#pragma unroll
      for (int w = 0; w < W; ++w) {
        s_digits[w * DIGITS + threadIdx.x] = at;
        at += count[w];
      }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kSortRounds; ++i)
      if (first + 64 * i + lane < last) s_pairs[mine[e[i] >> shift & (DIGITS - 1)] + rank[i]] = e[i];
    __syncthreads();
    if (pass + 1 < passes) {
#pragma unroll
      for (int i = 0; i < kSortRounds; ++i) {
        const int k = first + 64 * i + lane;
        if (k < last) e[i] = s_pairs[k];
      }
    }
  }
  for (int k = threadIdx.x; k < n; k += kSortThreads) {
    a.keys[k] = s_pairs[k] >> kPlaceBits;
    a.places[k] = s_pairs[k] & ((1u << kPlaceBits) - 1);
  }
}

// ---- sums ----------------------------------------------------------------------------------------------------------
struct SumArgs {
  const uint32_t *keys, *places;
  Range* ranges;   // [V], zeros
  int64_t rows;
  const void* dy;
  void* dw;
  float* parts;   // [piece][D], of pieces of one token
  int V, D, rows_per_group;
  float scale;
};
// N columns from c of the dy rows of the sorted places first, first + step, ...
template <typename T, int N> __device__ __forceinline__ vec<float, N> sum_places(const SumArgs& a, int64_t first, int64_t last, int step, int c) {
  vec<float, N> acc = fill_n<N>(0.f);
#pragma unroll 8
  for (int64_t k = first; k < last; k += step) acc += load_n<T, N>(static_cast<const T*>(a.dy) + (int64_t)a.places[k] * a.D + c);
  return acc;
}
// f(first column of a piece), a wave's sum of it, added over the waves, in their order, handed to `out` in wave 0
template <int N, typename F, typename G> __device__ __forceinline__ void over_waves(float* s_acc, int D, int first, int step, F&& f, G&& out) {   // pieces from `first`, 64 and then `step` on
  const int wave = wave_id(), lane = lane_id(), pieces = pieces_of<N>(D);
  for (int p0 = first; p0 < pieces; p0 += step) {
    const int i = p0 + lane, c = column<N>(i, D);
    vec<float, N> acc = fill_n<N>(0.f);
    if (i < pieces) acc = f(c);
    if (wave > 0)
#pragma unroll
      for (int e = 0; e < N; ++e) s_acc[((wave - 1) * N + e) * 64 + lane] = acc[e];
    __syncthreads();
    if (wave == 0 && i < pieces) {
#pragma unroll
      for (int w = 0; w < kWaves - 1; ++w)
#pragma unroll
        for (int e = 0; e < N; ++e) acc[e] += s_acc[(w * N + e) * 64 + lane];
      out(c, acc);
    }
    __syncthreads();
  }
}
template <typename T, int N> __global__ __launch_bounds__(kThreads) void run_sum_kernel(SumArgs a) {
  __shared__ float s_acc[(kWaves - 1) * N * 64];
  const int64_t piece = block_of_many(), first = piece * kRun, i = first + threadIdx.x;
  if (blockIdx.y == 0 && threadIdx.x < kRun && i < a.rows) {   // where a token ends and the next one begins
    const uint32_t k = a.keys[i], before = i > 0 ? a.keys[i - 1] : k + 1;
    if (k != before) {
      if (k < (uint32_t)a.V) a.ranges[k].first = (uint32_t)i;
      if (i > 0) a.ranges[before].end = (uint32_t)i;   // (keys behind the vocabulary are the last ones)
    }
    if (i == a.rows - 1 && k < (uint32_t)a.V) a.ranges[k].end = (uint32_t)a.rows;
  }
  if (first + kRun > a.rows) return;
  const uint32_t key = a.keys[first];
  if (key >= (uint32_t)a.V || a.keys[first + kRun - 1] != key) return;
  over_waves<N>(s_acc, a.D, 64 * blockIdx.y, 64 * gridDim.y, [&](int c) { return sum_places<T, N>(a, first + wave_id(), first + kRun, kWaves, c); },
                [&](int c, vec<float, N> v) { store_n<float, N>(a.parts + piece * a.D + c, v); });
}

constexpr int kMaxRowsPerGroup = 32, kFew = 8;   // kFew: tokens of a row that one wave, or part of one, sums by itself
// LPR: lanes to a row of few tokens, AT: pieces of each side by side, whose loads are on their way together (65536 tokens over 131072 rows of 2048 bf16: one by one 185 us, four 150)
template <typename T, int N, int LPR, int AT> __global__ __launch_bounds__(kThreads) void table_grad_kernel(SumArgs a) {
  __shared__ Range s_range[kMaxRowsPerGroup];
  __shared__ float s_acc[(kWaves - 1) * N * 64];
  // Rows G apart: the frequent tokens of a vocabulary stand together (a workgroup to 31 rows in a row: 162 us for 16384 tokens of 512 bf16 over 32000, the one of
  // the first tokens alone with all of it).
  const uint32_t G = gridDim.x * gridDim.z, first = (uint32_t)block_of_many();
  const int rows = (int)(((uint32_t)a.V - first + G - 1) / G), wave = wave_id();   // (none of a workgroup behind the last one)
  // (Bounds by a search of each workgroup among the keys: 14 trips to memory for 16384 tokens, 21 us instead of 16.)
  if ((int)threadIdx.x < rows) s_range[threadIdx.x] = a.ranges[first + threadIdx.x * G];
  __syncthreads();
  auto write = [&](int v, int c, vec<float, N> acc) { store_n<T, N>(static_cast<T*>(a.dw) + (int64_t)v * a.D + c, acc * a.scale); };
  for (int k = threadIdx.x / LPR; k < rows; k += kThreads / LPR) {
    const int64_t s = s_range[k].first, e = s_range[k].end;
    if (e - s > kFew) continue;
    for (int i = threadIdx.x % LPR; i < pieces_of<N>(a.D); i += AT * LPR) {
      vec<float, N> acc[AT];
      int c[AT];
#pragma unroll
      for (int u = 0; u < AT; ++u) {
        acc[u] = fill_n<N>(0.f);
        c[u] = column<N>(min(i + u * LPR, pieces_of<N>(a.D) - 1), a.D);
      }
#pragma unroll AT == 1 ? 8 : 2
      for (int64_t p = s; p < e; ++p) {
        const T* row = static_cast<const T*>(a.dy) + (int64_t)a.places[p] * a.D;
#pragma unroll
        for (int u = 0; u < AT; ++u) acc[u] += load_n<T, N>(row + c[u]);
      }
#pragma unroll
      for (int u = 0; u < AT; ++u)
        if (u == 0 || i + u * LPR < pieces_of<N>(a.D)) write(first + k * G, c[u], acc[u]);
    }
  }
  for (int k = 0; k < rows; ++k) {   // by all waves: places in front of the first whole piece, whole pieces, places behind
    const int64_t s = s_range[k].first, e = s_range[k].end;
    if (e - s <= kFew) continue;
    const int64_t c0 = (s + kRun - 1) / kRun, c1 = e / kRun;
    over_waves<N>(s_acc, a.D, 0, 64, [&](int c) {
      if (c1 <= c0) return sum_places<T, N>(a, s + wave, e, kWaves, c);
      vec<float, N> acc = sum_places<T, N>(a, s + wave, c0 * kRun, kWaves, c);
#pragma unroll 4
      for (int64_t p = c0 + wave; p < c1; p += kWaves) acc += load_n<float, N>(a.parts + p * a.D + c);
      return acc + sum_places<T, N>(a, c1 * kRun + wave, e, kWaves, c);
    }, [&](int c, vec<float, N> acc) { write(first + k * G, c, acc); });
  }
}

// f(type, std::integral_constant elements at a time)
template <typename F> int by_pieces(int dtype, int D, F&& f) {
  return by_tensor_type(dtype, [&](auto t) {
    using T = decltype(t);
    constexpr int N = elem_traits<T>::vec16;
    if (D >= N) return f(t, std::integral_constant<int, N>());
    return f(t, std::integral_constant<int, 1>());
  });
}
int launched() { return hipGetLastError() == hipSuccess ? 0 : -3; }

}  // namespace

int launch_embedding(const EmbeddingArgs& a, int dtype, hipStream_t stream) {
  return by_pieces(dtype, a.D, [&](auto t, auto n) {
    using T = decltype(t);
    auto go = [&](auto lpr) {
      constexpr int LPR = decltype(lpr)::value, rows = kThreads / LPR;
      hipLaunchKernelGGL((embedding_kernel<T, n.value, LPR>), many_blocks((a.tokens.rows + rows - 1) / rows), dim3(kThreads), 0, stream, a);
      return launched();
    };
    const int pieces = pieces_of<n.value>(a.D);
    if (pieces <= 16) return go(std::integral_constant<int, 16>());
    if (pieces <= 32) return go(std::integral_constant<int, 32>());
    return go(std::integral_constant<int, 64>());
  });
}

SortedGradPlan sorted_grad_plan(int64_t rows, int V, int D) {
  SortedGradPlan p = {};
  int bits = 1;
  while (bits < 31 && (int64_t)V >> bits != 0) ++bits;   // the keys are 0 .. V
  p.passes = (bits + 9) / 10;
  p.bits = (bits + p.passes - 1) / p.passes;
  p.together = rows <= kSortTokens && bits <= 18;
  if (p.together) {   // (the counts of sixteen waves lie in LDS)
    p.passes = bits <= 9 ? 1 : 2;
    p.bits = bits > 9 && bits <= 16 ? 8 : 9;
  }
  // 256 tokens to a wave until there are 256 workgroups, whose counts each of them adds up
  const int64_t waves = std::min<int64_t>(256 * kWaves, std::max<int64_t>(1, (rows + 255) / 256));
  p.wave_tokens = ((rows + waves - 1) / waves + 63) / 64 * 64;
  p.groups = (int)((rows + p.wave_tokens * kWaves - 1) / (p.wave_tokens * kWaves));
  p.rows_per_group = std::max(1, std::min(kMaxRowsPerGroup, V / 1024));
  auto bytes = [](int64_t n) { return (n + 255) / 256 * 256; };
  p.counts = bytes((int64_t)p.groups * (4 << p.bits));
  p.keys = bytes(4 * rows);
  p.places = bytes(4 * rows);
  p.parts = bytes(rows / kRun * D * 4);
  p.ranges = bytes((int64_t)V * sizeof(Range));
  p.total = p.counts + 2 * (p.keys + p.places) + p.parts + p.ranges;
  return p;
}

static int clearing_groups(int V) { return (int)(((int64_t)V + kClear - 1) / kClear); }
template <int BITS> static int launch_sort_all(const SortArgs& a, int passes, hipStream_t stream) {
  static PerDeviceOnce once;
  bool& configured = once.flag();
  constexpr int kBytes = (kSortTokens + (kSortThreads / 64 << BITS)) * 4;
  if (!configured) {
    if (hipFuncSetAttribute(reinterpret_cast<const void*>(&sort_all_kernel<BITS>), hipFuncAttributeMaxDynamicSharedMemorySize, kBytes) != hipSuccess) return -3;
    configured = true;
  }
  hipLaunchKernelGGL((sort_all_kernel<BITS>), dim3(1 + clearing_groups(a.V)), dim3(kSortThreads), kBytes, stream, a, passes);
  return launched();
}
int launch_sorted_grad(const SortedGradArgs& g, int dtype, hipStream_t stream) {
  const SortedGradPlan& p = g.plan;
  char* at = static_cast<char*>(g.workspace);
  auto take = [&](int64_t n) { char* r = at; at += n; return r; };
  uint32_t* const counts = reinterpret_cast<uint32_t*>(take(p.counts));
  uint32_t *keys[2], *places[2];
  for (int i = 0; i < 2; ++i) {
    keys[i] = reinterpret_cast<uint32_t*>(take(p.keys));
    places[i] = reinterpret_cast<uint32_t*>(take(p.places));
  }
  float* const parts = reinterpret_cast<float*>(take(p.parts));
  Range* const ranges = reinterpret_cast<Range*>(take(p.ranges));
  if (p.together) {
    const int last = (p.passes - 1) % 2;
    const SortArgs a = {g.tokens, g.V, g.padding, 0, p.bits, 0, nullptr, nullptr, keys[last], places[last], nullptr, ranges, 1};
    const int rc = p.bits == 8 ? launch_sort_all<8>(a, p.passes, stream) : launch_sort_all<9>(a, p.passes, stream);
    if (rc != 0) return rc;
  }
  for (int pass = 0; pass < p.passes && !p.together; ++pass) {
    const int to = pass % 2;
    const SortArgs a = {g.tokens, g.V, g.padding, pass * p.bits, p.bits, p.wave_tokens, pass > 0 ? keys[1 - to] : nullptr, pass > 0 ? places[1 - to] : nullptr,
                        keys[to], places[to], counts, ranges, p.groups};
    hipLaunchKernelGGL(sort_count_kernel, dim3(p.groups + (pass == 0 ? clearing_groups(g.V) : 0)), dim3(kThreads), 4 << p.bits, stream, a);
    hipLaunchKernelGGL(sort_place_kernel, dim3(p.groups), dim3(kThreads), kWaves * 4 << p.bits, stream, a);
  }
  const int sorted = (p.passes - 1) % 2;
  const SumArgs s = {keys[sorted], places[sorted], ranges, g.tokens.rows, g.dy, g.dw, parts, g.V, g.D, p.rows_per_group, g.scale};
  return by_pieces(dtype, g.D, [&](auto t, auto n) {
    using T = decltype(t);
    const int pieces = pieces_of<n.value>(g.D);
    hipLaunchKernelGGL((run_sum_kernel<T, n.value>), many_blocks((s.rows + kRun - 1) / kRun, std::min(8, (pieces + 63) / 64)), dim3(kThreads), 0, stream, s);
    const dim3 grid = many_blocks(((int64_t)g.V + p.rows_per_group - 1) / p.rows_per_group);
    if (pieces <= 16) hipLaunchKernelGGL((table_grad_kernel<T, n.value, 16, 1>), grid, dim3(kThreads), 0, stream, s);
    else if (pieces <= 32) hipLaunchKernelGGL((table_grad_kernel<T, n.value, 32, 1>), grid, dim3(kThreads), 0, stream, s);
    else if (pieces <= 64) hipLaunchKernelGGL((table_grad_kernel<T, n.value, 64, 1>), grid, dim3(kThreads), 0, stream, s);
    else hipLaunchKernelGGL((table_grad_kernel<T, n.value, 64, 4>), grid, dim3(kThreads), 0, stream, s);
    return launched();
  });
}

}  // namespace castle
