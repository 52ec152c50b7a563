// The norms on both sides of a residual sum: behind a block, with a gate and a scale, and in front of the next block.
//
//   n = x / sqrt(mean(x^2) + eps) w        y = residual + scale gate n        h = y / sqrt(mean(y^2) + eps) next_w
//
// y stays in 32 bits between the sum and the norm.  With xh = x / rms(x), yh = y / rms(y), c = scale w and q = c gate xh, the backward pass is
//   d  = dy + (dh next_w - yh mean(dh next_w yh)) / rms(y)      the gradient of y, and of the residual
//   dx = (c gate d - xh mean(d q)) / rms(x)       dgate = c d xh
//   dw = scale P,  dscale = w P  with P = sum over rows of gate d xh           dnext_w = sum over rows of dh yh
// so one column sum serves weight and scale, and mean(d q) follows from sums over dy q, dh next_w q and yh q: a row is summed over once.
//
// Bound by HBM: forward reads two tensors and writes two, backward reads four and writes two (the residual is read again rather than y: y is needed in 32 bits).  A row belongs to 16, 32 or
// 64 lanes, of more than 1024 elements to four or eight waves; a lane owns 8 columns of each piece of a row, so column sums stay in its registers over all its rows.
// us and TB/s: 65536 x 2048 with a gate of each sequence forward 213 and 5.0, backward 334 and 4.8, the join of the workgroups' column sums 9; 16384 x 512 14.6, 23.7 and 4.9 (4.6 and 4.2 TB/s).
#include "castle_tiles.h"
#include "castle_dispatch.h"
#include "castle_residual.h"
#include <algorithm>

namespace castle {
namespace {

template <typename T> using any8 = vec<T, 8> __attribute__((aligned(1)));
typedef vec<float, 8> vf;

constexpr int kForwardGroups = 1024;  // workgroups of the forward pass, at most
constexpr int kGateRows = 8;          // rows of a unit under a gate that several rows have

// LPR lanes of WPR waves have a row, NP pieces of 8 elements a lane
template <int LPR_, int WPR_, int NP_> struct Layout {
  static constexpr int LPR = LPR_, WPR = WPR_, NP = NP_, kBlock = WPR == 1 ? kThreads : 64 * WPR, kRows = kBlock / (LPR * WPR);
  // workgroups that a CU holds of the backward pass, and waves of a SIMD: all of a launch run at once, each over several rows (65536 x 2048 with a gate of each sequence: 1024 workgroups of which 768 ran at once 396 us, 764 of them 334)
  static constexpr int kHeld = WPR == 8 ? 1 : NP == 1 ? 3 : 2, kWavesPerSimd = WPR == 8 ? 2 : kHeld;
};
// workgroups for n turns, `most` at once, with as many turns each as they can have alike
int even_groups(int64_t n, int64_t most) {
  const int64_t turns = (n + most - 1) / most;
  return (int)((n + turns - 1) / turns);
}

template <typename T> __device__ __forceinline__ vec<T, 8> read8(const T* p, int left) {
  vec<T, 8> x = {};
  if (left >= 8) return *reinterpret_cast<const any8<T>*>(p);
#pragma unroll
  for (int e = 0; e < 8; ++e)
    if (e < left) x[e] = p[e];
  return x;
}
template <typename T> __device__ __forceinline__ void write8(T* p, vf v, int left) {
  const vec<T, 8> x = __builtin_convertvector(v, decltype(x));
  if (left >= 8) {
    *reinterpret_cast<any8<T>*>(p) = x;
    return;
  }
#pragma unroll
  for (int e = 0; e < 8; ++e)
    if (e < left) p[e] = x[e];
}
template <typename T> __device__ __forceinline__ vf wide(vec<T, 8> x) { return __builtin_convertvector(x, vf); }

// which of the workgroup's rows a lane has a part in: the same for a wave where a row is a wave's or more, and known to be
template <typename L> __device__ __forceinline__ int row_of_lane() {
  if constexpr (L::WPR > 1) return 0;
  else if constexpr (L::LPR == 64) return wave_id();
  else return threadIdx.x / L::LPR;
}
// sums over the lanes of a row, N at a time; `turn` alternates between two places in LDS, so that one barrier is enough
template <typename L, int N> __device__ __forceinline__ void row_sums(float (&v)[N], float* s, int& turn) {
#pragma unroll
  for (int o = 1; o < L::LPR; o <<= 1)
#pragma unroll
    for (int k = 0; k < N; ++k) v[k] += __shfl_xor(v[k], o);
  if constexpr (L::WPR > 1) {
    float* p = s + turn * (4 * L::WPR);
    turn ^= 1;
    if (lane_id() == 0)
#pragma unroll
      for (int k = 0; k < N; ++k) p[k * L::WPR + wave_id()] = v[k];
    __syncthreads();
#pragma unroll
    for (int k = 0; k < N; ++k) {
      v[k] = 0.f;
#pragma unroll
      for (int w = 0; w < L::WPR; ++w) v[k] += p[k * L::WPR + w];
    }
  }
}

// scale times w, and next_w, of this lane's columns
template <typename T, typename L> __device__ __forceinline__ void columns(const ResidualArgs& a, int sub, vf (&c)[L::NP], vec<T, 8> (&next)[L::NP]) {
#pragma unroll
  for (int p = 0; p < L::NP; ++p) {
    const int at = 8 * (p * L::LPR * L::WPR + sub), left = a.D - at;
#pragma unroll
    for (int e = 0; e < 8; ++e) c[p][e] = 1.f;
    if (a.w != nullptr) c[p] = wide<T>(read8(static_cast<const T*>(a.w) + at, left));
    if (a.scale != nullptr) c[p] *= wide<T>(read8(static_cast<const T*>(a.scale) + at, left));
    next[p] = {};
    if (a.next_w != nullptr) next[p] = read8(static_cast<const T*>(a.next_w) + at, left);
  }
}

template <typename T, typename L> __global__ __launch_bounds__(L::kBlock) void residual_kernel(ResidualArgs a) {
  __shared__ float s[8 * L::WPR];
  constexpr int TPR = L::LPR * L::WPR;
  const int sub = threadIdx.x % TPR;
  int turn = 0;
  vf c[L::NP];
  vec<T, 8> next[L::NP];
  columns<T, L>(a, sub, c, next);
  const int64_t step = (int64_t)gridDim.x * L::kRows;
  // the next row is requested before the one that is there is summed over
  vec<T, 8> nx[L::NP], nr[L::NP], ng[L::NP];
  auto fetch = [&](int64_t row) __attribute__((always_inline)) {
    const int64_t at = row * a.D;
#pragma unroll
    for (int p = 0; p < L::NP; ++p) {
      const int i = 8 * (p * TPR + sub), left = a.D - i;
      nx[p] = read8(static_cast<const T*>(a.x) + at + i, left);
      nr[p] = read8(static_cast<const T*>(a.residual) + at + i, left);
      if (a.gate != nullptr) ng[p] = read8(static_cast<const T*>(a.gate) + row / a.span * a.D + i, left);
    }
  };
  int64_t row = (int64_t)blockIdx.x * L::kRows + row_of_lane<L>();
  if (row < a.rows) fetch(row);
  for (; row < a.rows; row += step) {
    const int64_t at = row * a.D;
    vf x[L::NP], y[L::NP], g[L::NP];
#pragma unroll
    for (int p = 0; p < L::NP; ++p) {
      x[p] = wide<T>(nx[p]);
      y[p] = wide<T>(nr[p]);
      g[p] = wide<T>(ng[p]);
    }
    if (row + step < a.rows) fetch(row + step);
    float inv = 1.f;
    if (a.w != nullptr) {
      float sum[1] = {0.f};
#pragma unroll
      for (int p = 0; p < L::NP; ++p)
#pragma unroll
        for (int e = 0; e < 8; ++e) sum[0] = __builtin_fmaf(x[p][e], x[p][e], sum[0]);
      row_sums<L>(sum, s, turn);
      inv = 1.f / sqrtf(sum[0] / (float)a.D + a.eps);
    }
    float sum[1] = {0.f};
#pragma unroll
    for (int p = 0; p < L::NP; ++p) {
      vf q = x[p] * inv * c[p];
      if (a.gate != nullptr) q *= g[p];
      y[p] += q;
      const int i = 8 * (p * TPR + sub);
      write8<T>(static_cast<T*>(a.y) + at + i, y[p], a.D - i);
#pragma unroll
      for (int e = 0; e < 8; ++e) sum[0] = i + e < a.D ? __builtin_fmaf(y[p][e], y[p][e], sum[0]) : sum[0];
    }
    if (a.next_w != nullptr) {
      row_sums<L>(sum, s, turn);
      const float inv_y = 1.f / sqrtf(sum[0] / (float)a.D + a.eps);
#pragma unroll
      for (int p = 0; p < L::NP; ++p) {
        const int i = 8 * (p * TPR + sub);
        write8<T>(static_cast<T*>(a.h) + at + i, y[p] * inv_y * wide<T>(next[p]), a.D - i);
      }
      if (sub == 0 && a.next_rstd != nullptr) a.next_rstd[row] = inv_y;
    }
    if (sub == 0 && a.rstd != nullptr) a.rstd[row] = inv;
  }
}

// A unit is some rows one behind the other under one gate: those of a whole span, or part of it, whose sum over rows is then left in `unit_sums`.
struct Units {
  int64_t units, per_span, rows;   // rows of a unit, at most
};
struct BwdKernelArgs {
  ResidualBwdArgs b;
  Units u;
  float* parts;       // [workgroup][2][D]: P and the sums of dnext
  float* unit_sums;   // [unit][D], or nullptr: a unit has a whole span
};
// GATES: 0 none, 1 each row one of its own, 2 one of several rows.  BOTH: there are a norm of x and a gradient of h.  Without one of them its terms are left out, not multiplied by a zero: what the row
// holds may be infinite or NaN.  (By itself: the conditions cost the other one registers.)
template <typename T, typename L, int GATES, bool BOTH> __global__ __launch_bounds__(L::kBlock, L::kWavesPerSimd) void residual_bwd_kernel(BwdKernelArgs k) {
  const ResidualBwdArgs& b = k.b;
  const ResidualArgs& a = b.f;
  __shared__ float s[8 * L::WPR];
  extern __shared__ float s_columns[];   // [2][D]
  constexpr int TPR = L::LPR * L::WPR;
  const int sub = threadIdx.x % TPR;
  int turn = 0;
  vf c[L::NP], sum_p[L::NP], sum_next[L::NP], sum_unit[GATES == 2 ? L::NP : 1];
  vec<T, 8> next_w[L::NP];
  columns<T, L>(a, sub, c, next_w);
#pragma unroll
  for (int p = 0; p < L::NP; ++p) sum_p[p] = sum_next[p] = vf{};
  const float per = 1.f / (float)a.D;
  const bool with_x = BOTH || a.w != nullptr, with_h = BOTH || b.dh != nullptr;
  const int64_t step = (int64_t)gridDim.x * L::kRows;
  // a row of a unit; rows are requested one ahead
  struct Place { int64_t unit, row, last; };
  auto begin = [&](int64_t unit) __attribute__((always_inline)) {
    if constexpr (GATES != 2) return Place{unit, unit, unit + 1};
    const int64_t span = unit / k.u.per_span, first = span * a.span + unit % k.u.per_span * k.u.rows;
    return Place{unit, first, min(first + k.u.rows, (span + 1) * a.span)};
  };
  struct Row {
    vec<T, 8> x[L::NP], r[L::NP], dy[L::NP], dh[L::NP], g[GATES == 1 ? L::NP : 1];
    float inv, inv_y;
  };
  auto fetch = [&](int64_t row) __attribute__((always_inline)) {
    Row f;
    const int64_t at = row * a.D;
#pragma unroll
    for (int p = 0; p < L::NP; ++p) {
      const int i = 8 * (p * TPR + sub), left = a.D - i;
      f.x[p] = read8(static_cast<const T*>(a.x) + at + i, left);
      f.r[p] = read8(static_cast<const T*>(a.residual) + at + i, left);
      f.dy[p] = f.dh[p] = {};
      if (b.dy != nullptr) f.dy[p] = read8(static_cast<const T*>(b.dy) + at + i, left);
      if (b.dh != nullptr) f.dh[p] = read8(static_cast<const T*>(b.dh) + at + i, left);
      if constexpr (GATES == 1) f.g[p] = read8(static_cast<const T*>(a.gate) + at + i, left);
    }
    f.inv = with_x ? a.rstd[row] : 1.f;
    f.inv_y = with_h ? a.next_rstd[row] : 0.f;
    return f;
  };
  Place now = {(int64_t)blockIdx.x * L::kRows + row_of_lane<L>(), 0, 0};
  Row ahead;
  bool new_unit = true;
  vec<T, 8> unit_g[GATES == 2 ? L::NP : 1];
  if (now.unit < k.u.units) {
    now = begin(now.unit);
    ahead = fetch(now.row);
  }
  while (now.unit < k.u.units) {
    const int64_t row = now.row, unit = now.unit, at = row * a.D;
    const bool unit_ends = row + 1 == now.last;
    const Row f = ahead;
    if constexpr (GATES == 2)
      if (new_unit) {
#pragma unroll
        for (int p = 0; p < L::NP; ++p) {
          const int i = 8 * (p * TPR + sub);
          unit_g[p] = read8(static_cast<const T*>(a.gate) + row / a.span * a.D + i, a.D - i);
          sum_unit[p] = vf{};
        }
      }
    if (unit_ends) {
      now.unit += step;
      if (now.unit < k.u.units) now = begin(now.unit);
    } else {
      ++now.row;
    }
    new_unit = unit_ends;
    if (now.unit < k.u.units) ahead = fetch(now.row);
    const vec<T, 8>* g = GATES == 1 ? f.g : unit_g;
    float sum[4] = {};   // of dn yh, dy q, dn q, yh q
#pragma unroll
    for (int p = 0; p < L::NP; ++p) {
      vf q = wide<T>(f.x[p]) * f.inv * c[p];
      if constexpr (GATES != 0) q *= wide<T>(g[p]);
      const vf yh = (wide<T>(f.r[p]) + q) * f.inv_y, dn = wide<T>(f.dh[p]) * wide<T>(next_w[p]), d = wide<T>(f.dy[p]);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        sum[0] = __builtin_fmaf(dn[e], yh[e], sum[0]);
        sum[1] = __builtin_fmaf(d[e], q[e], sum[1]);
        sum[2] = __builtin_fmaf(dn[e], q[e], sum[2]);
        sum[3] = __builtin_fmaf(yh[e], q[e], sum[3]);
      }
    }
    row_sums<L>(sum, s, turn);
    const float m2 = sum[0] * per, m1 = (with_h ? sum[1] + f.inv_y * (sum[2] - m2 * sum[3]) : sum[1]) * per;
#pragma unroll
    for (int p = 0; p < L::NP; ++p) {
      const int i = 8 * (p * TPR + sub), left = a.D - i;
      const vf xh = wide<T>(f.x[p]) * f.inv;
      vf cg = c[p];
      if constexpr (GATES != 0) cg *= wide<T>(g[p]);
      const vf yh = (wide<T>(f.r[p]) + xh * cg) * f.inv_y, dhp = wide<T>(f.dh[p]), dn = dhp * wide<T>(next_w[p]);
      vf d = wide<T>(f.dy[p]);
      if (with_h) d += (dn - yh * m2) * f.inv_y;
      const vf t = d * xh;
      sum_next[p] += dhp * yh;
      if constexpr (GATES == 2) sum_unit[p] += t;
      else if constexpr (GATES == 1) sum_p[p] += t * wide<T>(g[p]);
      else sum_p[p] += t;
      if (b.dresidual != nullptr) write8<T>(static_cast<T*>(b.dresidual) + at + i, d, left);
      if (b.dx != nullptr) write8<T>(static_cast<T*>(b.dx) + at + i, with_x ? (d * cg - xh * m1) * f.inv : d * cg, left);
      if constexpr (GATES == 1)
        if (b.dgate != nullptr) write8<T>(static_cast<T*>(b.dgate) + at + i, t * c[p], left);
      if constexpr (GATES == 2)
        if (unit_ends) {
          sum_p[p] += sum_unit[p] * wide<T>(g[p]);
          if (b.dgate != nullptr && k.unit_sums == nullptr) write8<T>(static_cast<T*>(b.dgate) + row / a.span * a.D + i, sum_unit[p] * c[p], left);
          if (b.dgate != nullptr && k.unit_sums != nullptr) write8<float>(k.unit_sums + unit * a.D + i, sum_unit[p], left);
        }
    }
  }
  if (k.parts == nullptr) return;
  float* out = k.parts + (int64_t)blockIdx.x * 2 * a.D;
  if constexpr (L::WPR > 1) {
#pragma unroll
    for (int p = 0; p < L::NP; ++p) {
      const int i = 8 * (p * TPR + sub);
      write8<float>(out + i, sum_p[p], a.D - i);
      write8<float>(out + a.D + i, sum_next[p], a.D - i);
    }
  } else {
#pragma unroll
    for (int p = 0; p < L::NP; ++p)
#pragma unroll
      for (int e = 0; e < 8; ++e)
#pragma unroll
        for (int o = L::LPR; o < 64; o <<= 1) {
          sum_p[p][e] += __shfl_xor(sum_p[p][e], o);
          sum_next[p][e] += __shfl_xor(sum_next[p][e], o);
        }
    for (int w = 0; w < kThreads / 64; ++w) {
      if (wave_id() == w && lane_id() < L::LPR) {
#pragma unroll
        for (int p = 0; p < L::NP; ++p)
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const int i = 8 * (p * TPR + sub) + e;
            if (i >= a.D) continue;
            s_columns[i] = (w ? s_columns[i] : 0.f) + sum_p[p][e];
            s_columns[a.D + i] = (w ? s_columns[a.D + i] : 0.f) + sum_next[p][e];
          }
      }
      __syncthreads();
    }
    for (int i = threadIdx.x; i < 2 * a.D; i += kThreads) out[i] = s_columns[i];
  }
}

// Sums over the workgroups' parts: 16 columns of a workgroup, 16 threads down each; and, behind those, over the units of each gate.
struct JoinArgs {
  ResidualBwdArgs b;
  const float *parts, *unit_sums;
  int groups;
  int64_t per_span;
  int column_groups;   // workgroups of the columns of one of P and dnext; 0: none are wanted
};
template <typename T> __global__ __launch_bounds__(kThreads) void residual_join_kernel(JoinArgs a) {
  __shared__ float s[16][17];
  const int D = a.b.f.D, c = threadIdx.x % 16, r = threadIdx.x / 16;
  int64_t block = block_of_many();
  const float* from;
  int64_t count, stride;
  int col, which;
  const int64_t firsts = 2 * (int64_t)a.column_groups;
  int64_t gate = 0;
  if (block < firsts) {
    which = (int)(block / a.column_groups);
    col = (int)(block % a.column_groups) * 16 + c;
    from = a.parts + (int64_t)which * D;
    count = a.groups;
    stride = 2 * (int64_t)D;
  } else {
    const int64_t per_row = (D + 15) / 16;
    block -= firsts;
    gate = block / per_row;
    if (a.unit_sums == nullptr || gate >= a.b.f.rows / a.b.f.span) return;   // (of the whole workgroup)
    which = 2;
    col = (int)(block % per_row) * 16 + c;
    from = a.unit_sums + gate * a.per_span * D;
    count = a.per_span;
    stride = D;
  }
  float v = 0.f;
  if (col < D) {
#pragma unroll 8
    for (int64_t g = r; g < count; g += 16) v += from[g * stride + col];
  }
  s[r][c] = v;
  __syncthreads();
  if (r != 0 || col >= D) return;
#pragma unroll
  for (int k = 1; k < 16; ++k) v += s[k][c];
  const float w = a.b.f.w != nullptr ? (float)static_cast<const T*>(a.b.f.w)[col] : 1.f, scale = a.b.f.scale != nullptr ? (float)static_cast<const T*>(a.b.f.scale)[col] : 1.f;
  if (which == 2) {
    static_cast<T*>(a.b.dgate)[gate * D + col] = (T)(v * (w * scale));
  } else if (which == 1) {
    if (a.b.dnext != nullptr) static_cast<T*>(a.b.dnext)[col] = (T)v;
  } else {
    if (a.b.dw != nullptr) static_cast<T*>(a.b.dw)[col] = (T)(v * scale);
    if (a.b.dscale != nullptr) static_cast<T*>(a.b.dscale)[col] = (T)(v * w);
  }
}

// f(layout) for rows of D elements
template <typename F> int by_width(int D, F&& f) {
  if (D <= 128) return f(Layout<16, 1, 1>());
  if (D <= 256) return f(Layout<32, 1, 1>());
  if (D <= 512) return f(Layout<64, 1, 1>());
  if (D <= 1024) return f(Layout<64, 1, 2>());
  if (D <= 2048) return f(Layout<64, 4, 1>());
  if (D <= 4096) return f(Layout<64, 8, 1>());
  return D <= kResidualMaxWidth ? f(Layout<64, 8, 2>()) : -2;
}
int rows_of_group(int D) { return by_width(D, [](auto l) { return decltype(l)::kRows; }); }
int groups_at_once(int D) { return by_width(D, [](auto l) { return 256 * decltype(l)::kHeld; }); }
Units units_of(const ResidualBwdArgs& b) {
  const ResidualArgs& a = b.f;
  if (a.gate == nullptr || a.span == 1) return {a.rows, a.rows, 1};
  const int64_t lanes = (int64_t)groups_at_once(a.D) * rows_of_group(a.D);
  const int64_t rows = std::min(a.span, std::max<int64_t>(kGateRows, (a.rows + lanes - 1) / lanes)), per_span = (a.span + rows - 1) / rows;
  return {a.rows / a.span * per_span, per_span, rows};
}
int groups_of(const ResidualBwdArgs& b, const Units& u) {
  const int per = rows_of_group(b.f.D);
  return even_groups((u.units + per - 1) / per, groups_at_once(b.f.D));
}
bool wants_columns(const ResidualBwdArgs& b) { return b.dw != nullptr || b.dscale != nullptr || b.dnext != nullptr; }
bool wants_units(const ResidualBwdArgs& b, const Units& u) { return b.dgate != nullptr && b.f.span > 1 && u.per_span > 1; }
int64_t parts_bytes(const ResidualBwdArgs& b, const Units& u) { return wants_columns(b) ? ((int64_t)groups_of(b, u) * 2 * b.f.D * 4 + 255) / 256 * 256 : 0; }

}  // namespace

int64_t residual_bwd_workspace(const ResidualBwdArgs& b) {
  const Units u = units_of(b);
  return parts_bytes(b, u) + (wants_units(b, u) ? u.units * b.f.D * 4 : 0);
}

int launch_residual(const ResidualArgs& a, int dtype, hipStream_t stream) {
  return by_tensor_type(dtype, [&](auto t) {
    using T = decltype(t);
    return by_width(a.D, [&](auto l) {
      using L = decltype(l);
      const int groups = even_groups((a.rows + L::kRows - 1) / L::kRows, kForwardGroups);
      hipLaunchKernelGGL((residual_kernel<T, L>), dim3(groups), dim3(L::kBlock), 0, stream, a);
      return hipGetLastError() == hipSuccess ? 0 : -3;
    });
  });
}

int launch_residual_bwd(const ResidualBwdArgs& b, int dtype, void* workspace, hipStream_t stream) {
  const Units u = units_of(b);
  const int groups = groups_of(b, u);
  const bool with_columns = wants_columns(b), with_units = wants_units(b, u);
  BwdKernelArgs k = {b, u, with_columns ? static_cast<float*>(workspace) : nullptr, with_units ? reinterpret_cast<float*>(static_cast<char*>(workspace) + parts_bytes(b, u)) : nullptr};
  if (b.f.gate == nullptr || b.f.span == 1) k.b.f.span = b.f.rows;   // (one unit of each row)
  int rc = by_tensor_type(dtype, [&](auto t) {
    using T = decltype(t);
    return by_width(b.f.D, [&](auto l) {
      using L = decltype(l);
      const size_t lds = L::WPR == 1 && with_columns ? 2 * (size_t)b.f.D * 4 : 0;
      const dim3 grid(groups), block(L::kBlock);
      auto go = [&](auto both_) {
        constexpr bool BOTH = decltype(both_)::value;
        if (b.f.gate == nullptr) hipLaunchKernelGGL((residual_bwd_kernel<T, L, 0, BOTH>), grid, block, lds, stream, k);
        else if (b.f.span == 1) hipLaunchKernelGGL((residual_bwd_kernel<T, L, 1, BOTH>), grid, block, lds, stream, k);
        else hipLaunchKernelGGL((residual_bwd_kernel<T, L, 2, BOTH>), grid, block, lds, stream, k);
        return hipGetLastError() == hipSuccess ? 0 : -3;
      };
      return b.f.w != nullptr && b.dh != nullptr ? go(std::true_type()) : go(std::false_type());
    });
  });
  if (rc != 0 || (!with_columns && !with_units)) return rc;
  const int64_t per_row = (b.f.D + 15) / 16;
  const JoinArgs j = {b, k.parts, k.unit_sums, groups, u.per_span, with_columns ? (int)per_row : 0};
  const int64_t blocks = 2 * (int64_t)j.column_groups + (with_units ? b.f.rows / b.f.span * per_row : 0);
  return by_tensor_type(dtype, [&](auto t) {
    hipLaunchKernelGGL((residual_join_kernel<decltype(t)>), many_blocks(blocks), dim3(kThreads), 0, stream, j);
    return hipGetLastError() == hipSuccess ? 0 : -3;
  });
}

}  // namespace castle
