// Gated feed-forward block:  u = x w_in^T, (g, v) the halves of u's columns, h = act(g) v, y = h w_out^T
//   dh = dy w_out     dg = dh v act'(g)     dv = dh act(g)     dx = [dg dv] w_in     dw_in = [dg dv]^T x     dw_out = dy^T h
#include "castle_tiles.h"
#include "castle_dispatch.h"
#include "castle_gated.h"
#include "castle_gelu.h"
#include "castle_gemm.h"
#include "castle_rows.h"
#include <algorithm>

namespace castle {
namespace {

typedef vec<float, 8> vf;

// act(g) and its derivative
template <typename T, int ACT> struct Gate {
  float act, slope;
  __device__ __forceinline__ explicit Gate(float g) {
    if constexpr (ACT == kSilu) {
      const float s = sizeof(T) == 4 ? 1.f / (1.f + expf(-g)) : sigmoid_l2(g * kLog2e);
      act = g * s;
      slope = __builtin_fmaf(act, 1.f - s, s);
    } else {
      const Normal<T> n(g);
      act = g * n.cdf;
      slope = __builtin_fmaf(g * 0.3989422804f, n.e, n.cdf);
    }
  }
};

// h of u = [R][2 F]; BWD: [dg dv] of dh and u, in place of u or not, and h
template <typename T, int ACT> __global__ __launch_bounds__(kThreads) void gate_kernel(const T* u, int64_t n, int F, T* h) {
  const int64_t i = (block_of_many() * kThreads + threadIdx.x) * 8, row = i / F, col = i - row * F;
  if (i >= n) return;
  const vf g = __builtin_convertvector((frag<T>)*reinterpret_cast<const frag_mem<T>*>(u + row * 2 * F + col), vf);
  const vf v = __builtin_convertvector((frag<T>)*reinterpret_cast<const frag_mem<T>*>(u + row * 2 * F + F + col), vf);
  vf y;
#pragma unroll
  for (int e = 0; e < 8; ++e) y[e] = Gate<T, ACT>(g[e]).act * v[e];
  *reinterpret_cast<frag_mem<T>*>(h + i) = __builtin_convertvector(y, frag<T>);
}
template <typename T, int ACT> __global__ __launch_bounds__(kThreads) void gate_bwd_kernel(const T* u, const T* dh, int64_t n, int F, T* du, T* h) {
  const int64_t i = (block_of_many() * kThreads + threadIdx.x) * 8, row = i / F, col = i - row * F;
  if (i >= n) return;
  const vf g = __builtin_convertvector((frag<T>)*reinterpret_cast<const frag_mem<T>*>(u + row * 2 * F + col), vf);
  const vf v = __builtin_convertvector((frag<T>)*reinterpret_cast<const frag_mem<T>*>(u + row * 2 * F + F + col), vf);
  const vf d = __builtin_convertvector((frag<T>)*reinterpret_cast<const frag_mem<T>*>(dh + i), vf);
  vf dg, dv, y;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const Gate<T, ACT> a(g[e]);
    dg[e] = d[e] * (v[e] * a.slope);
    dv[e] = d[e] * a.act;
    y[e] = a.act * v[e];
  }
  *reinterpret_cast<frag_mem<T>*>(du + row * 2 * F + col) = __builtin_convertvector(dg, frag<T>);
  *reinterpret_cast<frag_mem<T>*>(du + row * 2 * F + F + col) = __builtin_convertvector(dv, frag<T>);
  if (h != nullptr) *reinterpret_cast<frag_mem<T>*>(h + i) = __builtin_convertvector(y, frag<T>);
}

int64_t up(int64_t n) { return (n + 255) / 256 * 256; }
int elem_size(int dtype) { return dtype == 0 ? 4 : 2; }

struct Operand2 {
  const void* p;
  int64_t ld;
  bool kc;   // contraction-contiguous
};
int64_t product_workspace(int M, int N, int K, int dtype) { return up(gemm_workspace(M, N, K, elem_size(dtype), false)); }
int product(const Operand2& a, const Operand2& b, void* c, int M, int N, int K, int dtype, void* workspace, hipStream_t stream) {
  const GemmArgs g = {a.p, b.p, c, nullptr, M, N, K, a.ld, b.ld, N, kGemmPlain, 0, nullptr, nullptr, nullptr, 0, 1, nullptr, 0.f, nullptr, nullptr};
  return launch_gemm(g, a.kc, b.kc, dtype, static_cast<float*>(workspace), stream);
}
// Both gradients of a projection y = x w^T, dy [R][N], x [R][K], in one launch where that is ahead
int64_t grads_bytes(int R, int N, int K, int dtype, bool dw, bool dx) {
  const int64_t both = dw && dx ? grads_workspace(R, N, K, elem_size(dtype), kGemmPlain, false) : -1;
  if (both >= 0) return up(both);
  return std::max(dw ? product_workspace(N, K, R, dtype) : 0, dx ? product_workspace(R, K, N, dtype) : 0);
}
int grads(const Operand2& dy, const Operand2& x, const Operand2& w, void* dw, void* dx, int R, int N, int K, int dtype, void* workspace, hipStream_t stream) {
  if (dw != nullptr && dx != nullptr && grads_workspace(R, N, K, elem_size(dtype), kGemmPlain, false) >= 0) {
    GradsArgs p = {};
    p.w = {dy.p, x.p, dw, nullptr, N, K, R, dy.ld, x.ld, K, kGemmPlain, 0, nullptr, nullptr, nullptr, 0, 1, nullptr, 0.f, nullptr, nullptr};
    p.x = {dy.p, w.p, dx, nullptr, R, K, N, dy.ld, w.ld, K, kGemmPlain, 0, nullptr, nullptr, nullptr, 0, 1, nullptr, 0.f, nullptr, nullptr};
    return launch_grads(p, dtype, static_cast<float*>(workspace), nullptr, stream);
  }
  if (dx != nullptr)
    if (const int rc = product({dy.p, dy.ld, true}, {w.p, w.ld, false}, dx, R, K, N, dtype, workspace, stream)) return rc;
  return dw == nullptr ? 0 : product({dy.p, dy.ld, false}, {x.p, x.ld, false}, dw, N, K, R, dtype, workspace, stream);
}

template <typename F> int by_type_and_act(int dtype, int act, F&& f) {
  return by_tensor_type(dtype, [&](auto t) {
    return act == kSilu ? f(t, std::integral_constant<int, kSilu>()) : f(t, std::integral_constant<int, kGeluGate>());
  });
}

}  // namespace

// state: u
int64_t gated_state(int R, int D, int F, int dtype) { return up((int64_t)R * 2 * F * elem_size(dtype)); }
int64_t gated_workspace(int R, int D, int F, int dtype, bool keeps) {
  return up((int64_t)R * F * elem_size(dtype)) + (keeps ? 0 : gated_state(R, D, F, dtype)) + std::max(product_workspace(R, 2 * F, D, dtype), product_workspace(R, D, F, dtype));
}
int launch_gated(const GatedArgs& a, void* y, void* state, int dtype, void* workspace, hipStream_t stream) {
  char* at = static_cast<char*>(workspace);
  void* h = at;
  at += up((int64_t)a.R * a.F * elem_size(dtype));
  void* u = state;
  if (u == nullptr) {
    u = at;
    at += gated_state(a.R, a.D, a.F, dtype);
  }
  if (const int rc = product({a.x, a.ld_x, true}, {a.w_in, a.ld_in, true}, u, a.R, 2 * a.F, a.D, dtype, at, stream)) return rc;
  const int64_t n = (int64_t)a.R * a.F;
  const int rc = by_type_and_act(dtype, a.act, [&](auto t, auto act) {
    using T = decltype(t);
    hipLaunchKernelGGL((gate_kernel<T, decltype(act)::value>), many_blocks((n / 8 + kThreads - 1) / kThreads), dim3(kThreads), 0, stream, static_cast<const T*>(u), n, a.F, static_cast<T*>(h));
    return hipGetLastError() == hipSuccess ? 0 : -3;
  });
  return rc != 0 ? rc : product({h, a.F, true}, {a.w_out, a.ld_out, true}, y, a.R, a.D, a.F, dtype, at, stream);
}

int64_t gated_bwd_workspace(int R, int D, int F, int dtype, int gradients) {
  const bool dx = gradients & 1, dw_in = gradients & 2, dw_out = gradients & 4;
  const int64_t hidden = up((int64_t)R * F * elem_size(dtype));
  return (dw_out ? hidden : 0) + hidden + gated_state(R, D, F, dtype) +
         std::max({product_workspace(R, F, D, dtype), dw_out ? product_workspace(D, F, R, dtype) : 0, grads_bytes(R, 2 * F, D, dtype, dw_in, dx)});
}
int launch_gated_bwd(const GatedArgs& a, const void* dy, const void* state, void* dx, void* dw_in, void* dw_out, int dtype, void* workspace, hipStream_t stream) {
  char* at = static_cast<char*>(workspace);
  const int64_t hidden = up((int64_t)a.R * a.F * elem_size(dtype)), n = (int64_t)a.R * a.F;
  auto take = [&](int64_t bytes) { char* p = at; at += bytes; return p; };
  void *h = dw_out != nullptr ? take(hidden) : nullptr, *dh = take(hidden), *du = take(gated_state(a.R, a.D, a.F, dtype));
  if (const int rc = product({dy, a.D, true}, {a.w_out, a.ld_out, false}, dh, a.R, a.F, a.D, dtype, at, stream)) return rc;
  int rc = by_type_and_act(dtype, a.act, [&](auto t, auto act) {
    using T = decltype(t);
    hipLaunchKernelGGL((gate_bwd_kernel<T, decltype(act)::value>), many_blocks((n / 8 + kThreads - 1) / kThreads), dim3(kThreads), 0, stream, static_cast<const T*>(state),
                       static_cast<const T*>(dh), n, a.F, static_cast<T*>(du), static_cast<T*>(h));
    return hipGetLastError() == hipSuccess ? 0 : -3;
  });
  if (rc != 0) return rc;
  if (dw_out != nullptr && (rc = product({dy, a.D, false}, {h, a.F, false}, dw_out, a.D, a.F, a.R, dtype, at, stream)) != 0) return rc;
  return grads({du, 2 * a.F, true}, {a.x, a.ld_x, true}, {a.w_in, a.ld_in, true}, dw_in, dx, a.R, 2 * a.F, a.D, dtype, at, stream);
}

}  // namespace castle
