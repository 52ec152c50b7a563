// A step of AdamW over many tensors and the norm of their gradients.
//
//   g' = c g, c = min(1, max_norm / (norm + 1e-6))      m = b1 m + (1 - b1) g'        v = b2 v + (1 - b2) g'^2
//   p = p (1 - lr wd) - lr / (1 - b1^t) m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// States of 8 bits: 256 elements share 2^E, the least power of two with which the largest of them is at most 448, and are e4m3 numbers times that: m, and r = sqrt(v), whose
// range is half of v's in octaves.  They are rounded up or down by chance, so that the mean is kept.  To the nearest, a state would stay where it is: a step with b2 = 0.999 moves r by
// 0.05 %, steps of e4m3 are 6 to 12 %.  A second moment that is not zero stays above zero (2^-18 of the largest): as zero its element would move by lr m / eps.  16-bit
// parameters are rounded by chance too where there is a seed: lr = 1e-4 moves none of bf16 to the nearest.
// Numbers are formed by single 32-bit operations, rounded each (no contraction), in the order of the formulas; the quotient of a step is off by an ulp or two, and so are roots but for those of 8-bit
// states beside 32-bit parameters.
//
// Bound by HBM: per element of 16 bits 10 bytes with states of 8 bits, 22 with 32, 28 of fp32, and the gradients once more for their norm, which has to be there before the first element.
// us and TB/s: 65M bf16 numbers with states of 32 bits 267 and 5.3, the norm before 42 and 3.1 (of gradients that no writes precede 28 and 4.6); 318M with states of 8 bits 665 and 4.8, where a
// quarter of the time is instructions (Philox, exponents, e4m3 and back), the norm 142 and 4.5; 2.1M of fp32 12.4, the norm and its join 8.
// Tensors go 64 to a launch of the step and 192 to one of the norm, their addresses in its arguments: a table in memory would have to be written anew for every step, as gradients move.
#include "castle_tiles.h"
#include "castle_dispatch.h"
#include "castle_optim.h"
#include "castle_philox.h"
#include <algorithm>

namespace castle {
namespace {

constexpr int kGroup = kThreads * 8;      // elements of a workgroup's turn, eight a thread
constexpr int kTurns = 4;                 // turns of a workgroup
constexpr int kWaves = kThreads / 64;

// rows of any alignment (gfx950 reads and writes them at the speed of aligned ones where they are aligned)
template <typename T> using any8 = vec<T, 8> __attribute__((aligned(1)));

struct LaunchTensors {
  OptimTensor t[kTensorsOfLaunch];
  uint32_t first[kTensorsOfLaunch];   // piece (kGroup * kTurns elements) that each begins with; behind the last tensor the number of pieces
  int count, number;                  // number: of the first tensor, in the whole call
};
static_assert(sizeof(LaunchTensors) + 64 <= 4096, "arguments of a launch");

// the tensor that a piece lies in: every lane looks at one of them
__device__ __forceinline__ int tensor_of(const LaunchTensors& a, uint32_t piece) {
  const int i = min(lane_id(), a.count - 1);
  const uint64_t begun = __ballot(lane_id() < a.count && a.first[i] <= piece);
  return 63 - __builtin_clzll(begun);   // (one without elements has a piece too, so firsts grow)
}

template <typename T> __device__ __forceinline__ vec<T, 8> raw8(const T* p, int left) {
  vec<T, 8> x = {};
  if (left >= 8) {
    x = *reinterpret_cast<const any8<T>*>(p);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (e < left) x[e] = p[e];
  }
  return x;
}
template <typename T> __device__ __forceinline__ void write8(T* p, vec<T, 8> x, int left) {
  if (left >= 8) {
    *reinterpret_cast<any8<T>*>(p) = x;
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (e < left) p[e] = x[e];
  }
}

// ---- norm ----------------------------------------------------------------------------------------------------------
// Sums of squares in double: of the largest floats they do not overflow, of the smallest they do not vanish, and the adds (two instructions an element) hide behind the reads.  The next piece is
// requested before the one that is there is added up.
constexpr int kGradsOfLaunch = 192;
struct LaunchGrads {
  const void* g[kGradsOfLaunch];
  int64_t n[kGradsOfLaunch];
  uint32_t first[kGradsOfLaunch];   // piece that each begins with
  int count;
};
static_assert(sizeof(LaunchGrads) + 64 <= 4096, "arguments of a launch");
template <typename T> __global__ __launch_bounds__(kThreads) void norm_parts_kernel(LaunchGrads a, uint32_t pieces, double* parts) {
  __shared__ double s[kWaves];
  double sum[2] = {0, 0};
  vec<T, 8> x[2][kTurns];
  auto fetch = [&](int slot, uint32_t piece) __attribute__((always_inline)) {
    const int lane = lane_id();
    int k = 0;
#pragma unroll
    for (int i = 0; i < kGradsOfLaunch; i += 64) k += __popcll(__ballot(i + lane < a.count && a.first[min(i + lane, a.count - 1)] <= piece));
    k = __builtin_amdgcn_readfirstlane(k - 1);
    const int64_t begin = (int64_t)(piece - a.first[k]) * (kGroup * kTurns) + threadIdx.x * 8;
#pragma unroll
    for (int j = 0; j < kTurns; ++j) {
      const int64_t left = a.n[k] - begin - j * kGroup;
      x[slot][j] = raw8(static_cast<const T*>(a.g[k]) + begin + j * kGroup, (int)max((int64_t)0, min((int64_t)8, left)));
    }
  };
  auto add = [&](int slot) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < kTurns; ++j)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const double g = (double)(float)x[slot][j][e];
        sum[e & 1] = __builtin_fma(g, g, sum[e & 1]);
      }
  };
  uint32_t piece = blockIdx.x;
  fetch(0, piece);
  while (true) {
    if (piece + gridDim.x < pieces) fetch(1, piece + gridDim.x);
    add(0);
    if ((piece += gridDim.x) >= pieces) break;
    if (piece + gridDim.x < pieces) fetch(0, piece + gridDim.x);
    add(1);
    if ((piece += gridDim.x) >= pieces) break;
  }
  double v = sum[0] + sum[1];
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) v += __shfl_xor(v, o);
  if (lane_id() == 0) s[wave_id()] = v;
  __syncthreads();
  if (threadIdx.x == 0) {
#pragma unroll
    for (int w = 1; w < kWaves; ++w) v += s[w];
    parts[blockIdx.x] = v;
  }
}

// One workgroup: the norm of `parts` partial sums (if there are any), and the numbers of a step (if one follows)
__global__ __launch_bounds__(1024) void begin_kernel(const double* parts, int count, float* norm, StepOptions o, StepNumbers* numbers) {
#pragma clang fp contract(off)
  __shared__ double s[16];
  double v = 0;
  for (int i = threadIdx.x; i < count; i += 1024) v += parts[i];
#pragma unroll
  for (int k = 1; k < 64; k <<= 1) v += __shfl_xor(v, k);
  if (lane_id() == 0) s[wave_id()] = v;
  __syncthreads();
  if (threadIdx.x != 0) return;
  float n = 0.f;
  if (parts != nullptr) {
    for (int w = 1; w < 16; ++w) v += s[w];
    n = (float)sqrt(v);
    *norm = n;
  } else if (norm != nullptr) {
    n = *norm;
  }
  if (numbers == nullptr) return;
  StepNumbers r = {};
  const int64_t t = *o.step + 1;
  *o.step = t;
  const double lr = o.lr_device != nullptr ? (double)*o.lr_device : o.lr;
  r.clip = 1.f;
  if (o.max_norm >= 0) {
    const float c = (float)o.max_norm / (n + 1e-6f);
    r.clip = c > 1.f ? 1.f : c;   // (a NaN stays one)
  }
  r.rate = (float)(lr / (1 - pow(o.b1, (double)t)));
  r.root = (float)(1 / sqrt(1 - pow(o.b2, (double)t)));
  r.keep = (float)(1 - lr * o.weight_decay);
  r.step = (uint32_t)t;
  *numbers = r;
}

// ---- step ----------------------------------------------------------------------------------------------------------
__device__ __forceinline__ float power_of_two(int e) { return __builtin_bit_cast(float, (uint32_t)(e + 127) << 23); }
__device__ __forceinline__ uint32_t bits_of(float x) { return __builtin_bit_cast(uint32_t, x); }

// Roots and quotients to an ulp or two: correctly rounded ones took a fifth of the kernel with states of 8 bits.  The instruction takes denormal numbers for zero: where one of a wave's is, those are
// scaled before it.  Zero has the root zero; `least`, the bits of 2^-126, where eps is zero: then 2^-63, and the element stays where it is.
__device__ __forceinline__ bool denormal(float x) { return __builtin_amdgcn_classf(x, 0x90); }
__device__ __forceinline__ void fast_roots(const vec<float, 8>& v, uint32_t least, vec<float, 8>& r) {
  bool scaled = false;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    r[e] = __builtin_amdgcn_sqrtf(__builtin_bit_cast(float, max(bits_of(v[e]), least)));   // (as whole numbers, of which a NaN is among the largest)
    scaled |= denormal(v[e]);
  }
  if (__ballot(scaled) == 0) return;
#pragma unroll
  for (int e = 0; e < 8; ++e)
    if (denormal(v[e])) r[e] = __builtin_amdgcn_sqrtf(v[e] * 0x1p64f) * 0x1p-32f;
}

// Eight numbers to e4m3, up or down by chance: the instruction adds the upper bits of its last operand to what it cuts off, below the normal numbers too, which is what castle_hip.h says (its results
// are those of that formula for 1.7e7 numbers from 2^-20 to 448 and all that is not finite).
__device__ __forceinline__ vec<uint8_t, 8> to_e4m3(const vec<float, 8>& x, const Words& u) {
  vec<uint32_t, 2> c = {};
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    int w = 0;
    w = __builtin_amdgcn_cvt_sr_fp8_f32(x[4 * k], u.w[2 * k] << 16, w, 0);
    w = __builtin_amdgcn_cvt_sr_fp8_f32(x[4 * k + 1], u.w[2 * k] & 0xffff0000u, w, 1);
    w = __builtin_amdgcn_cvt_sr_fp8_f32(x[4 * k + 2], u.w[2 * k + 1] << 16, w, 2);
    c[k] = __builtin_amdgcn_cvt_sr_fp8_f32(x[4 * k + 3], u.w[2 * k + 1] & 0xffff0000u, w, 3);
  }
  typedef vec<uint8_t, 8> v8;
  return __builtin_bit_cast(v8, c);
}
__device__ __forceinline__ vec<float, 8> from_e4m3(vec<uint8_t, 8> codes, float power) {
  typedef vec<uint32_t, 2> v2;
  const v2 c = __builtin_bit_cast(v2, codes);
  vec<float, 8> x;
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)c[k], false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)c[k], true);
    x[4 * k] = lo[0] * power;
    x[4 * k + 1] = lo[1] * power;
    x[4 * k + 2] = hi[0] * power;
    x[4 * k + 3] = hi[1] * power;
  }
  return x;
}
// the largest |x| of 256 elements, 32 lanes of them, as bits; SIGNED: some may be negative, FINITE: of those that are finite
template <bool SIGNED, bool FINITE> __device__ __forceinline__ uint32_t largest(const vec<float, 8>& x) {
  uint32_t most = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const uint32_t b = SIGNED || FINITE ? bits_of(x[e]) & 0x7fffffff : bits_of(x[e]);
    most = max(most, !FINITE || b < 0x7f800000u ? b : 0u);
  }
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) most = max(most, (uint32_t)__shfl_xor((int)most, o));
  return most;
}
template <bool SIGNED> __device__ __forceinline__ uint32_t largest_finite(const vec<float, 8>& x) {
  uint32_t most = largest<SIGNED, false>(x);
  if (__ballot(most >= 0x7f800000u) != 0) most = largest<SIGNED, true>(x);   // (of the whole wave: its lanes exchange)
  return most;
}
// E for the bits of the largest
__device__ __forceinline__ int exponent_of(uint32_t most) { return min(max((int)(most >> 23) - 135 + ((most & 0x7fffff) > 0x600000), -126), 120); }

// eight 16-bit parameters by chance
template <typename T> __device__ __forceinline__ vec<T, 8> by_chance(const vec<float, 8>& q, const Words& r) {
  vec<T, 8> y;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float p = q[e];
    const bool finite = __builtin_isfinite(p);
    const uint32_t bits = bits_of(p), u = finite ? half_of(r, e) : 0;   // (what is not finite has nothing to be cut off)
    if constexpr (__is_same(T, bf16_t)) {
      y[e] = __builtin_bit_cast(bf16_t, (uint16_t)((bits + u) >> 16));
    } else {
#pragma clang fp contract(off)
      const float up = __builtin_bit_cast(float, (bits + (u >> 3)) & 0xffffe000u);
      const float low = copysignf(floorf(fabsf(p) * 0x1p24f + (float)u * 0x1p-16f) * 0x1p-24f, p);
      y[e] = (T)(finite ? fabsf(p) < 0x1p-14f ? low : up : p);
    }
  }
  return y;
}

// SMALL: states of 8 bits; CHANCE: 16-bit parameters are rounded by chance
template <typename T, bool SMALL, bool CHANCE> __global__ __launch_bounds__(kThreads) void adamw_kernel(LaunchTensors a, const StepNumbers* numbers, const int64_t* seed,
                                                                                                       float b1, float c1, float b2, float c2, float eps) {
#pragma clang fp contract(off)
  typedef vec<float, 8> vf;
  typedef std::conditional_t<SMALL, uint8_t, float> State;
  const int k = __builtin_amdgcn_readfirstlane(tensor_of(a, blockIdx.x));
  const OptimTensor t = a.t[k];
  const StepNumbers s = *numbers;
  const uint32_t least = eps == 0.f ? bits_of(0x1p-126f) : 0;
  const uint64_t key = SMALL || CHANCE ? (uint64_t)*seed : 0, at_step = (uint64_t)(uint32_t)(a.number + k) << 32 | s.step;
  const int64_t begin = (int64_t)(blockIdx.x - a.first[k]) * (kGroup * kTurns) + threadIdx.x * 8;
  // what a turn reads is requested a turn ahead
  struct Turn {
    vec<T, 8> g, p;
    vec<State, 8> m, v;
    float pm, pv;
  };
  auto left_at = [&](int64_t at) __attribute__((always_inline)) { return (int)max((int64_t)0, min((int64_t)8, t.n - at)); };
  auto fetch = [&](int64_t at) __attribute__((always_inline)) {
    const int left = left_at(at);
    Turn r;
    r.g = raw8(static_cast<const T*>(t.g) + at, left);
    r.p = raw8(static_cast<const T*>(t.p) + at, left);
    r.m = raw8(static_cast<const State*>(t.m) + at, left);
    r.v = raw8(static_cast<const State*>(t.v) + at, left);
    if constexpr (SMALL) {
      r.pm = left > 0 ? power_of_two(t.em[at / kScaleBlock]) : 1.f;
      r.pv = left > 0 ? power_of_two(t.ev[at / kScaleBlock]) : 1.f;
    }
    return r;
  };
  if (begin - 8 * lane_id() >= t.n) return;   // (of a wave: 256 elements exchange their maximum)
  Turn next = fetch(begin);
#pragma unroll 1
  for (int j = 0; j < kTurns; ++j) {
    const int64_t at = begin + j * kGroup;
    const int left = left_at(at);
    const Turn now = next;
    const bool more = j + 1 < kTurns && at + kGroup - 8 * lane_id() < t.n;
    if (more) next = fetch(at + kGroup);
    const vf x = __builtin_convertvector(now.g, vf), p = __builtin_convertvector(now.p, vf);
    vf m, v, r, q;
    if constexpr (SMALL) {
      m = from_e4m3(now.m, now.pm);
      v = from_e4m3(now.v, now.pv);
      v *= v;
    } else {
      m = now.m;
      v = now.v;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float g = x[e] * s.clip;
      m[e] = b1 * m[e] + c1 * g;
      v[e] = b2 * v[e] + c2 * (g * g);
    }
    // (correctly rounded beside parameters of 32 bits: a root that is one unit off is rounded to another state in one of 6 million cases, and those show where parameters keep their 24 bits)
    if constexpr (SMALL && sizeof(T) == 4) {
#pragma unroll
      for (int e = 0; e < 8; ++e) r[e] = sqrtf(v[e]);
    } else {
      fast_roots(v, least, r);
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) q[e] = p[e] * s.keep - s.rate * m[e] * fast_rcp(r[e] * s.root + eps);
    const uint64_t counter = 4 * (uint64_t)(at >> 3);
    if constexpr (SMALL) {
      // (the largest root is that of the largest square: the exponent goes by the correctly rounded one)
      const int em = exponent_of(largest_finite<true>(m)), ev = exponent_of(bits_of(sqrtf(__builtin_bit_cast(float, largest_finite<false>(v)))));
      m *= power_of_two(-em);
      r *= power_of_two(-ev);
#pragma unroll
      for (int e = 0; e < 8; ++e) r[e] = v[e] == 0.f ? 0.f : __builtin_bit_cast(float, max(bits_of(r[e]), bits_of(0x1p-9f)));   // what is not zero stays above it
      const vec<uint8_t, 8> cv = to_e4m3(r, philox(counter, key, at_step)), cm = to_e4m3(m, philox(counter + 1, key, at_step));
      write8<uint8_t>(static_cast<uint8_t*>(t.m) + at, cm, left);
      write8<uint8_t>(static_cast<uint8_t*>(t.v) + at, cv, left);
      if (left > 0 && at % kScaleBlock == 0) {
        t.em[at / kScaleBlock] = (int8_t)em;
        t.ev[at / kScaleBlock] = (int8_t)ev;
      }
    } else {
      write8<float>(static_cast<float*>(t.m) + at, m, left);
      write8<float>(static_cast<float*>(t.v) + at, v, left);
    }
    vec<T, 8> y;
    if constexpr (CHANCE) y = by_chance<T>(q, philox(counter + 2, key, at_step));
    else y = __builtin_convertvector(q, decltype(y));
    write8<T>(static_cast<T*>(t.p) + at, y, left);
    if (!more) return;
  }
}

// One without elements has a piece in which there is nothing to do.  (All elements of a call are at most 2^36: of 256 threads a piece, 2^31 threads.)
uint32_t pieces_of(int64_t n) { return (uint32_t)std::max<int64_t>(1, (n + kGroup * kTurns - 1) / (kGroup * kTurns)); }
// f(tensors of a launch, their pieces) for 64 of them at a time; a tensor's number is its place in the call.
template <typename F> int for_launches(const OptimTensor* tensors, int count, F&& f) {
  for (int from = 0; from < count; from += kTensorsOfLaunch) {
    LaunchTensors a = {};
    a.count = std::min(count - from, kTensorsOfLaunch);
    a.number = from;
    uint32_t pieces = 0;
    for (int i = 0; i < a.count; ++i) {
      a.t[i] = tensors[from + i];
      a.first[i] = pieces;
      pieces += pieces_of(a.t[i].n);
    }
    if (const int rc = f(a, pieces)) return rc;
  }
  return 0;
}

}  // namespace

int64_t optim_workspace(int count) { return 256 + (int64_t)((count + kGradsOfLaunch - 1) / kGradsOfLaunch) * kNormGroups * 8; }

static int norm_parts(const OptimTensor* tensors, int count, int dtype, double* parts, int* made, hipStream_t stream) {
  *made = 0;
  for (int from = 0; from < count; from += kGradsOfLaunch) {
    LaunchGrads a = {};
    a.count = std::min(count - from, kGradsOfLaunch);
    uint32_t pieces = 0;
    for (int i = 0; i < a.count; ++i) {
      a.g[i] = tensors[from + i].g;
      a.n[i] = tensors[from + i].n;
      a.first[i] = pieces;
      pieces += pieces_of(a.n[i]);
    }
    const int groups = (int)std::min<uint32_t>(pieces, kNormGroups);
    const int rc = by_tensor_type(dtype, [&](auto t) {
      hipLaunchKernelGGL((norm_parts_kernel<decltype(t)>), dim3(groups), dim3(kThreads), 0, stream, a, pieces, parts + *made);
      return hipGetLastError() == hipSuccess ? 0 : -3;
    });
    if (rc != 0) return rc;
    *made += groups;
  }
  return 0;
}

int launch_grad_norm(const OptimTensor* tensors, int count, float* norm, int dtype, void* workspace, hipStream_t stream) {
  double* parts = reinterpret_cast<double*>(static_cast<char*>(workspace) + 256);
  int made = 0;
  if (const int rc = norm_parts(tensors, count, dtype, parts, &made, stream)) return rc;
  hipLaunchKernelGGL(begin_kernel, dim3(1), dim3(1024), 0, stream, parts, made, norm, StepOptions{}, nullptr);
  return hipGetLastError() == hipSuccess ? 0 : -3;
}

int launch_adamw(const OptimTensor* tensors, int count, const StepOptions& o, float* norm, bool clip_here, int dtype, void* workspace, hipStream_t stream) {
  StepNumbers* numbers = static_cast<StepNumbers*>(workspace);
  double* parts = nullptr;
  int made = 0;
  if (clip_here) {
    parts = reinterpret_cast<double*>(static_cast<char*>(workspace) + 256);
    if (const int rc = norm_parts(tensors, count, dtype, parts, &made, stream)) return rc;
  }
  hipLaunchKernelGGL(begin_kernel, dim3(1), dim3(1024), 0, stream, parts, made, norm, o, numbers);
  if (hipGetLastError() != hipSuccess) return -3;
  const float b1 = (float)o.b1, c1 = (float)(1 - o.b1), b2 = (float)o.b2, c2 = (float)(1 - o.b2), eps = (float)o.eps;
  return for_launches(tensors, count, [&](const LaunchTensors& a, uint32_t pieces) {
    return by_tensor_type(dtype, [&](auto t) {
      using T = decltype(t);
      auto go = [&](auto small, auto chance) {
        hipLaunchKernelGGL((adamw_kernel<T, decltype(small)::value, decltype(chance)::value>), dim3(pieces), dim3(kThreads), 0, stream, a, numbers, o.seed, b1, c1, b2, c2, eps);
        return hipGetLastError() == hipSuccess ? 0 : -3;
      };
      const std::true_type yes;
      const std::false_type no;
      const bool small = tensors[0].em != nullptr;
      if constexpr (sizeof(T) == 4) return small ? go(yes, no) : go(no, no);
      else return small ? go(yes, yes) : o.seed != nullptr ? go(no, yes) : go(no, no);
    });
  });
}

}  // namespace castle
