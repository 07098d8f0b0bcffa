// norm_backward.hip -- the gradients of CliffordLayerNorm (the forward: norm.hip,
// holograph/layers/normalization.py:44-67).
//
// With y_i = gamma_i xh_i + beta_i (geometric products, gamma on the left), xh = x / rms and
// rms^2 = mean_i |x_i|^2 + 2 eps, for the gradient dy of y:
//   gx_i     = ~gamma_i dy_i              (the adjoint of the left product is the product with the reverse)
//   dx_i     = (gx_i - xh_i <gx, xh> / d) / rms        (+ the residual branch's gradient)
//   dgamma_i = sum over the tokens of dy_i ~xh_i
//   dbeta_i  = sum over the tokens of dy_i
// <gx, xh> is the sum over the token's multivectors of the inner products of their 8 values.
//
// Everything is computed in fp32; dx is rounded once to x's type.  dgamma and dbeta are sums over
// all tokens: every workgroup adds its tokens in order into a partial plane, and the planes are
// added in order, so results do not depend on scheduling.

#include <hip/hip_runtime.h>

#include "pauli_common.h"
#include "ygg_common.h"

namespace ygg {
namespace {

constexpr int kNbMaxD = 4096;     // the forward's limit
constexpr int kNbPlaneTokens = 64;  // tokens per partial plane

__device__ inline void load_mv(const float* p, size_t n, float v[8]) {
  const float4* q = reinterpret_cast<const float4*>(p + n * 8);
  const float4 a = q[0], b = q[1];
  v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
  v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
}
__device__ inline void load_mv(const uint16_t* p, size_t n, float v[8]) {
  const uint4 q = *reinterpret_cast<const uint4*>(p + n * 8);
  v[0] = bf_lo(q.x); v[1] = bf_hi(q.x); v[2] = bf_lo(q.y); v[3] = bf_hi(q.y);
  v[4] = bf_lo(q.z); v[5] = bf_hi(q.z); v[6] = bf_lo(q.w); v[7] = bf_hi(q.w);
}
__device__ inline void store_mv(float* p, size_t n, const float v[8]) {
  float4* q = reinterpret_cast<float4*>(p + n * 8);
  q[0] = make_float4(v[0], v[1], v[2], v[3]);
  q[1] = make_float4(v[4], v[5], v[6], v[7]);
}
__device__ inline void store_mv(uint16_t* p, size_t n, const float v[8]) {
  *reinterpret_cast<uint4*>(p + n * 8) =
      make_uint4(pack2_bf16(v[0], v[1]), pack2_bf16(v[2], v[3]), pack2_bf16(v[4], v[5]), pack2_bf16(v[6], v[7]));
}
__device__ constexpr float rev(int c) { return c >= 4 ? -1.f : 1.f; }  // grades 2 and 3 change sign

// o = (~)a b or a ~b, over the blades
template <bool REV_A, bool REV_B>
__device__ inline void product(const float a[8], const float b[8], float o[8]) {
#pragma unroll
  for (int c = 0; c < 8; ++c) {
    const int mc = blade_to_mask(c);
    float s = 0.f;
#pragma unroll
    for (int p = 0; p < 8; ++p) {
      const int mp = blade_to_mask(p), q = mask_to_blade(mp ^ mc);
      const float sign = (float)mask_product_sign(mp, mp ^ mc) * (REV_A ? rev(p) : 1.f) * (REV_B ? rev(q) : 1.f);
      s = __builtin_fmaf(sign * a[p], b[q], s);
    }
    o[c] = s;
  }
}

// One wave per token: 1 / rms and dx.
template <typename XT, typename GT>
__global__ __launch_bounds__(256) void norm_dx_kernel(const GT* __restrict__ dy, const XT* __restrict__ x, int N, int d,
                                                      const float* __restrict__ gamma, float two_eps,
                                                      const XT* __restrict__ residual, XT* __restrict__ dx,
                                                      float* __restrict__ rrms) {
  const int lane = threadIdx.x & 63;
  const int t = blockIdx.x * 4 + (threadIdx.x >> 6);
  if (t >= N) return;
  const size_t row = (size_t)t * d;
  float n2 = 0.f, dot = 0.f;
  for (int i = lane; i < d; i += 64) {
    float v[8], u[8], g[8], gx[8];
    load_mv(x, row + i, v);
    load_mv(dy, row + i, u);
    load_mv(gamma, i, g);
    product<true, false>(g, u, gx);
#pragma unroll
    for (int c = 0; c < 8; ++c) {
      n2 = __builtin_fmaf(v[c], v[c], n2);
      dot = __builtin_fmaf(gx[c], v[c], dot);
    }
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    n2 += __shfl_xor(n2, o);
    dot += __shfl_xor(dot, o);
  }
  const float r = 1.0f / sqrtf(n2 / (float)d + two_eps);
  const float w = dot * r * r / (float)d;  // <gx, x> / (rms^2 d): dx = (gx - x w) / rms
  if (lane == 0) rrms[t] = r;
  for (int i = lane; i < d; i += 64) {
    float v[8], u[8], g[8], gx[8], o[8];
    load_mv(x, row + i, v);
    load_mv(dy, row + i, u);
    load_mv(gamma, i, g);
    product<true, false>(g, u, gx);
#pragma unroll
    for (int c = 0; c < 8; ++c) o[c] = r * __builtin_fmaf(-w, v[c], gx[c]);
    if (residual != nullptr) {
      float s[8];
      load_mv(residual, row + i, s);
#pragma unroll
      for (int c = 0; c < 8; ++c) o[c] += s[c];
    }
    store_mv(dx, row + i, o);
  }
}

// Partial sums of dgamma and dbeta over kNbPlaneTokens tokens: a thread per multivector.
template <typename XT, typename GT>
__global__ __launch_bounds__(64) void norm_param_kernel(const GT* __restrict__ dy, const XT* __restrict__ x, int N, int d,
                                                        const float* __restrict__ rrms, float* __restrict__ part) {
  const int i = blockIdx.y * 64 + threadIdx.x;
  if (i >= d) return;
  const int t0 = blockIdx.x * kNbPlaneTokens, t1 = min(N, t0 + kNbPlaneTokens);
  float sg[8] = {}, sb[8] = {};
  for (int t = t0; t < t1; ++t) {
    float v[8], u[8], o[8];
    load_mv(x, (size_t)t * d + i, v);
    load_mv(dy, (size_t)t * d + i, u);
    const float r = rrms[t];
#pragma unroll
    for (int c = 0; c < 8; ++c) v[c] *= r;
    product<false, true>(u, v, o);
#pragma unroll
    for (int c = 0; c < 8; ++c) {
      sg[c] += o[c];
      sb[c] += u[c];
    }
  }
  float* p = part + ((size_t)blockIdx.x * d + i) * 16;
  store_mv(p, 0, sg);
  store_mv(p, 1, sb);
}

// The planes added in order: a thread per value.
__global__ __launch_bounds__(256) void norm_param_reduce_kernel(const float* __restrict__ part, int planes, int d,
                                                                float* __restrict__ dgamma, float* __restrict__ dbeta) {
  const int n = blockIdx.x * 256 + threadIdx.x;
  if (n >= d * 16) return;
  float s = 0.f;
  for (int p = 0; p < planes; ++p) s += part[(size_t)p * d * 16 + n];
  const int i = n >> 4, c = n & 15;
  (c < 8 ? dgamma : dbeta)[(size_t)i * 8 + (c & 7)] = s;
}

int planes_of(int N) { return (N + kNbPlaneTokens - 1) / kNbPlaneTokens; }
size_t rrms_bytes(int N) { return ((size_t)N * 4 + 255) / 256 * 256; }

template <typename XT, typename GT>
int launch(const void* dy, const void* x, int N, int d, const float* gamma, float two_eps, const void* residual,
           void* dx, float* dgamma, float* dbeta, void* workspace, hipStream_t stream) {
  float* rrms = static_cast<float*>(workspace);
  float* part = reinterpret_cast<float*>(static_cast<char*>(workspace) + rrms_bytes(N));
  if (N > 0) {
    hipLaunchKernelGGL((norm_dx_kernel<XT, GT>), dim3((N + 3) / 4), dim3(256), 0, stream, static_cast<const GT*>(dy),
                       static_cast<const XT*>(x), N, d, gamma, two_eps, static_cast<const XT*>(residual),
                       static_cast<XT*>(dx), rrms);
    if (check_launch("norm backward")) return -1;
    hipLaunchKernelGGL((norm_param_kernel<XT, GT>), dim3(planes_of(N), (d + 63) / 64), dim3(64), 0, stream,
                       static_cast<const GT*>(dy), static_cast<const XT*>(x), N, d, rrms, part);
    if (check_launch("norm backward (gamma and beta)")) return -1;
  }
  hipLaunchKernelGGL(norm_param_reduce_kernel, dim3((d * 16 + 255) / 256), dim3(256), 0, stream, part, planes_of(N), d,
                     dgamma, dbeta);
  return check_launch("norm backward (reduction)");
}

}  // namespace
}  // namespace ygg

using namespace ygg;

YGG_API size_t ygg_clifford_layer_norm_backward_workspace_bytes(int N, int d) {
  if (N < 0 || d < 1 || d > kNbMaxD) return 0;
  return rrms_bytes(N) + (size_t)planes_of(N) * d * 16 * sizeof(float);
}

YGG_API int ygg_clifford_layer_norm_backward(const void* dy, int dy_dtype, const void* x, int x_dtype, int N, int d,
                                             const float* gamma, double eps, const void* residual_grad, void* dx,
                                             float* dgamma, float* dbeta, void* workspace, size_t workspace_bytes,
                                             hipStream_t stream) {
  YGG_CHECK_ARG(x_dtype == kF32 || x_dtype == kBF16, "ygg_clifford_layer_norm_backward: x dtype %d unsupported", x_dtype);
  YGG_CHECK_ARG(dy_dtype == kF32 || dy_dtype == kBF16, "ygg_clifford_layer_norm_backward: dy dtype %d unsupported",
                dy_dtype);
  YGG_CHECK_ARG(N >= 0 && d >= 1 && d <= kNbMaxD, "ygg_clifford_layer_norm_backward: bad sizes N=%d d=%d (d <= %d)", N, d,
                kNbMaxD);
  YGG_CHECK_ARG(eps >= 0.0, "ygg_clifford_layer_norm_backward: eps must be non-negative");
  YGG_CHECK_ARG(gamma && dgamma && dbeta && (N == 0 || (dy && x && dx)),
                "ygg_clifford_layer_norm_backward: null pointer argument");
  const size_t need = ygg_clifford_layer_norm_backward_workspace_bytes(N, d);
  YGG_CHECK_ARG(need == 0 || (workspace && workspace_bytes >= need),
                "ygg_clifford_layer_norm_backward: workspace of %zu bytes, need %zu", workspace ? workspace_bytes : 0,
                need);
  const float two_eps = (float)(2.0 * eps);  // as the forward adds it
  if (x_dtype == kF32)
    return dy_dtype == kF32
               ? launch<float, float>(dy, x, N, d, gamma, two_eps, residual_grad, dx, dgamma, dbeta, workspace, stream)
               : launch<float, uint16_t>(dy, x, N, d, gamma, two_eps, residual_grad, dx, dgamma, dbeta, workspace, stream);
  return dy_dtype == kF32
             ? launch<uint16_t, float>(dy, x, N, d, gamma, two_eps, residual_grad, dx, dgamma, dbeta, workspace, stream)
             : launch<uint16_t, uint16_t>(dy, x, N, d, gamma, two_eps, residual_grad, dx, dgamma, dbeta, workspace,
                                          stream);
}
