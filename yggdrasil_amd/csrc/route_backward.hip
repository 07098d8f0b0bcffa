// route_backward.hip -- the gradient of the routing weights back to the logits and, for the
// grade-energy router, to the tokens and the router's parameters (the forward: route.hip,
// holograph/layers/clifford_router.py:54-104).
//
// The routing weights of a token are its chosen experts' probabilities over their sum, w_s =
// p_s / sum_j p_j: the softmax over the chosen logits alone (the forward's 1e-12 next to a sum of
// at least 1 / 64 is below half a step of fp32).  The choice itself has no gradient.  With g_s the
// gradient of w_s,
//   dl_s = w_s (g_s - sum_j w_j g_j)   for a chosen expert, 0 for every other
// For logits = share W^T + b with share_h = energy_h / (total + 1e-12), the energies summed over
// the blades of each grade:
//   dW[e] = sum_t dl_te share_t,  db[e] = sum_t dl_te,  ds_t = sum_e dl_te W[e]
//   denergy_h = (ds_h - <ds, share>) / (total + 1e-12),  dx = 2 x denergy_grade(x)
//
// Everything is computed in fp32; dx is rounded once to x's type.  The sums over the tokens are
// added in an order that the sizes alone fix.

#include <hip/hip_runtime.h>

#include "pauli_common.h"
#include "ygg_common.h"

namespace ygg {
namespace {

constexpr int kRbMaxExperts = 64, kRbMaxK = 8;

// dl of one token's slots: all lanes that call it with the same t get the same values
__device__ inline void slot_gradients(const float* __restrict__ w, const float* __restrict__ g, size_t t, int k,
                                      float* dl) {
  float dot = 0.f;
#pragma unroll
  for (int s = 0; s < kRbMaxK; ++s)
    if (s < k) dot = __builtin_fmaf(w[t * k + s], g[t * k + s], dot);
#pragma unroll
  for (int s = 0; s < kRbMaxK; ++s) dl[s] = s < k && k > 1 ? w[t * k + s] * (g[t * k + s] - dot) : 0.f;
}

// A thread per (token, expert): every logit's gradient written once.
__global__ __launch_bounds__(256) void route_backward_kernel(const int32_t* __restrict__ idx, const float* __restrict__ w,
                                                             const float* __restrict__ g, int N, int E, int k,
                                                             float* __restrict__ dlogits) {
  const size_t n = (size_t)blockIdx.x * 256 + threadIdx.x;
  if (n >= (size_t)N * E) return;
  const size_t t = n / E;
  const int e = (int)(n - t * E);
  float dl[kRbMaxK], v = 0.f;
  slot_gradients(w, g, t, k, dl);
#pragma unroll
  for (int s = 0; s < kRbMaxK; ++s)
    if (s < k && idx[t * k + s] == e) v += dl[s];
  dlogits[n] = v;
}

__device__ inline void load8(const float* p, size_t n, float v[8]) {
  const float4* q = reinterpret_cast<const float4*>(p + n * 8);
  const float4 a = q[0], b = q[1];
  v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
  v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
}
__device__ inline void load8(const uint16_t* p, size_t n, float v[8]) {
  const uint4 q = *reinterpret_cast<const uint4*>(p + n * 8);
  v[0] = bf_lo(q.x); v[1] = bf_hi(q.x); v[2] = bf_lo(q.y); v[3] = bf_hi(q.y);
  v[4] = bf_lo(q.z); v[5] = bf_hi(q.z); v[6] = bf_lo(q.w); v[7] = bf_hi(q.w);
}
__device__ inline void store8(float* p, size_t n, const float v[8]) {
  float4* q = reinterpret_cast<float4*>(p + n * 8);
  q[0] = make_float4(v[0], v[1], v[2], v[3]);
  q[1] = make_float4(v[4], v[5], v[6], v[7]);
}
__device__ inline void store8(uint16_t* p, size_t n, const float v[8]) {
  *reinterpret_cast<uint4*>(p + n * 8) =
      make_uint4(pack2_bf16(v[0], v[1]), pack2_bf16(v[2], v[3]), pack2_bf16(v[4], v[5]), pack2_bf16(v[6], v[7]));
}

// One wave per token: dx (plus add), and the token's energy shares for the parameters' sums.
template <typename T>
__global__ __launch_bounds__(256) void energy_backward_kernel(const T* __restrict__ x, int N, int d,
                                                              const float* __restrict__ W, int E, int k,
                                                              const int32_t* __restrict__ idx,
                                                              const float* __restrict__ w, const float* __restrict__ g,
                                                              const T* __restrict__ add, T* __restrict__ dx,
                                                              float* __restrict__ shares) {
  const int lane = threadIdx.x & 63;
  const int t = blockIdx.x * 4 + (threadIdx.x >> 6);
  if (t >= N) return;
  const size_t row = (size_t)t * d;
  float en[4] = {0.f, 0.f, 0.f, 0.f};
  for (int i = lane; i < d; i += 64) {
    float v[8];
    load8(x, row + i, v);
    en[0] = __builtin_fmaf(v[0], v[0], en[0]);
    en[3] = __builtin_fmaf(v[7], v[7], en[3]);
#pragma unroll
    for (int c = 0; c < 3; ++c) {
      en[1] = __builtin_fmaf(v[1 + c], v[1 + c], en[1]);
      en[2] = __builtin_fmaf(v[4 + c], v[4 + c], en[2]);
    }
  }
#pragma unroll
  for (int h = 0; h < 4; ++h)
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) en[h] += __shfl_xor(en[h], o);
  const float total = ((en[0] + en[1]) + (en[2] + en[3])) + 1e-12f;
  float dl[kRbMaxK], ds[4] = {0.f, 0.f, 0.f, 0.f}, sh[4], dot = 0.f;
  slot_gradients(w, g, t, k, dl);
#pragma unroll
  for (int s = 0; s < kRbMaxK; ++s) {
    const int e = s < k ? idx[(size_t)t * k + s] : 0;
    if (s < k && e >= 0 && e < E)
#pragma unroll
      for (int h = 0; h < 4; ++h) ds[h] = __builtin_fmaf(dl[s], W[e * 4 + h], ds[h]);
  }
#pragma unroll
  for (int h = 0; h < 4; ++h) {
    sh[h] = en[h] / total;
    dot = __builtin_fmaf(ds[h], sh[h], dot);
  }
  if (lane < 4) shares[(size_t)t * 4 + lane] = lane == 0 ? sh[0] : lane == 1 ? sh[1] : lane == 2 ? sh[2] : sh[3];
  float de[4];
#pragma unroll
  for (int h = 0; h < 4; ++h) de[h] = 2.f * (ds[h] - dot) / total;
  for (int i = lane; i < d; i += 64) {
    float v[8], o[8] = {};
    load8(x, row + i, v);
    if (add != nullptr) load8(add, row + i, o);
#pragma unroll
    for (int c = 0; c < 8; ++c) o[c] = __builtin_fmaf(v[c], de[c == 0 ? 0 : c < 4 ? 1 : c < 7 ? 2 : 3], o[c]);
    store8(dx, row + i, o);
  }
}

// One workgroup per expert: its slots of all tokens, added per thread and then over the threads.
__global__ __launch_bounds__(256) void router_param_kernel(const int32_t* __restrict__ idx, const float* __restrict__ w,
                                                           const float* __restrict__ g,
                                                           const float* __restrict__ shares, int N, int k,
                                                           float* __restrict__ dW, float* __restrict__ db) {
  const int e = blockIdx.x;
  float s5[5] = {0.f, 0.f, 0.f, 0.f, 0.f};
  for (int t = threadIdx.x; t < N; t += 256) {
    float v = 0.f;
    bool mine = false;
    for (int s = 0; s < k; ++s) mine |= idx[(size_t)t * k + s] == e;
    if (!mine) continue;
    float dl[kRbMaxK];
    slot_gradients(w, g, t, k, dl);
#pragma unroll
    for (int s = 0; s < kRbMaxK; ++s)
      if (s < k && idx[(size_t)t * k + s] == e) v += dl[s];
#pragma unroll
    for (int h = 0; h < 4; ++h) s5[h] = __builtin_fmaf(v, shares[(size_t)t * 4 + h], s5[h]);
    s5[4] += v;
  }
  __shared__ float red[4][5];
#pragma unroll
  for (int h = 0; h < 5; ++h) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) s5[h] += __shfl_xor(s5[h], o);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6][h] = s5[h];
  }
  __syncthreads();
  if (threadIdx.x < 5) {
    const float v = (red[0][threadIdx.x] + red[1][threadIdx.x]) + (red[2][threadIdx.x] + red[3][threadIdx.x]);
    if (threadIdx.x < 4) dW[e * 4 + threadIdx.x] = v;
    else db[e] = v;
  }
}

}  // namespace
}  // namespace ygg

using namespace ygg;

YGG_API int ygg_route_backward(const int32_t* topk_idx, const float* topk_w, const float* dtopk_w, int N, int E, int k,
                               float* dlogits, hipStream_t stream) {
  YGG_CHECK_ARG(N >= 0 && E >= 1 && E <= kRbMaxExperts && k >= 1 && k <= kRbMaxK && k <= E,
                "ygg_route_backward: bad sizes N=%d E=%d k=%d (E <= %d, k <= min(%d, E))", N, E, k, kRbMaxExperts, kRbMaxK);
  if (N == 0) return 0;
  YGG_CHECK_ARG(topk_idx && topk_w && dtopk_w && dlogits, "ygg_route_backward: null pointer argument");
  const size_t n = (size_t)N * E;
  hipLaunchKernelGGL(route_backward_kernel, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, stream, topk_idx, topk_w,
                     dtopk_w, N, E, k, dlogits);
  return check_launch("ygg_route_backward");
}

YGG_API size_t ygg_route_energy_backward_workspace_bytes(int N, int E) {
  if (N < 0 || E < 1) return 0;
  return (size_t)N * 16;
}

YGG_API int ygg_route_energy_backward(const void* x, int x_dtype, int N, int d, const float* router_w, int E, int k,
                                      const int32_t* topk_idx, const float* topk_w, const float* dtopk_w,
                                      const void* dx_add, void* dx, float* drouter_w, float* drouter_b, void* workspace,
                                      size_t workspace_bytes, hipStream_t stream) {
  YGG_CHECK_ARG(x_dtype == kF32 || x_dtype == kBF16, "ygg_route_energy_backward: x dtype %d unsupported", x_dtype);
  YGG_CHECK_ARG(N >= 0 && d >= 1 && E >= 1 && E <= kRbMaxExperts && k >= 1 && k <= kRbMaxK && k <= E,
                "ygg_route_energy_backward: bad sizes N=%d d=%d E=%d k=%d (E <= %d, k <= min(%d, E))", N, d, E, k,
                kRbMaxExperts, kRbMaxK);
  YGG_CHECK_ARG(drouter_w && drouter_b && (N == 0 || (x && router_w && topk_idx && topk_w && dtopk_w && dx)),
                "ygg_route_energy_backward: null pointer argument");
  const size_t need = ygg_route_energy_backward_workspace_bytes(N, E);
  YGG_CHECK_ARG(need == 0 || (workspace && workspace_bytes >= need),
                "ygg_route_energy_backward: workspace of %zu bytes, need %zu", workspace ? workspace_bytes : 0, need);
  float* shares = static_cast<float*>(workspace);
  if (N > 0) {
    const dim3 grid((N + 3) / 4);
    if (x_dtype == kF32)
      hipLaunchKernelGGL(energy_backward_kernel<float>, grid, dim3(256), 0, stream, static_cast<const float*>(x), N, d,
                         router_w, E, k, topk_idx, topk_w, dtopk_w, static_cast<const float*>(dx_add),
                         static_cast<float*>(dx), shares);
    else
      hipLaunchKernelGGL(energy_backward_kernel<uint16_t>, grid, dim3(256), 0, stream, static_cast<const uint16_t*>(x), N,
                         d, router_w, E, k, topk_idx, topk_w, dtopk_w, static_cast<const uint16_t*>(dx_add),
                         static_cast<uint16_t*>(dx), shares);
    if (check_launch("ygg_route_energy_backward")) return -1;
  }
  hipLaunchKernelGGL(router_param_kernel, dim3(E), dim3(256), 0, stream, topk_idx, topk_w, dtopk_w, shares, N, k,
                     drouter_w, drouter_b);
  return check_launch("ygg_route_energy_backward (parameters)");
}
