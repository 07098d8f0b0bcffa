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

#include <algorithm>

#include "rows.h"
#include "ygg_common.h"

namespace ygg {
namespace {

constexpr int kNbMaxD = 4096;     // the forward's limit
constexpr int kNbMaxN = 0x7fff0000;  // (the workgroups step past the last token by up to a batch each)
constexpr int kNbPlaneTokens = 64;  // tokens per partial plane

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

// dx of one token by a wave, which reads its row twice; returns 1 / rms.
template <typename XT, typename GT>
__device__ __forceinline__ float norm_dx_row(const GT* dy, const XT* x, size_t row, int d, const float* gamma,
                                             float two_eps, const XT* residual, XT* dx, int lane) {
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
  return r;
}

// One wave per token: 1 / rms and dx.
template <typename XT, typename GT>
__global__ __launch_bounds__(256) void norm_dx_kernel(const GT* __restrict__ dy, const XT* __restrict__ x, int N, int d,
                                                      const float* __restrict__ gamma, float two_eps, const XT* residual,
                                                      XT* dx, float* __restrict__ rrms) {
  const int lane = threadIdx.x & 63;
  const int t = blockIdx.x * 4 + (threadIdx.x >> 6);
  if (t >= N) return;
  const float r = norm_dx_row(dy, x, (size_t)t * d, d, gamma, two_eps, residual, dx, lane);
  if (lane == 0) rrms[t] = r;
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

// ---- rows of at most 1024 multivectors: one pass -------------------------------------------------
// A workgroup of four waves takes U tokens at a time: CS waves share a row (a lane holds NQ of its multivectors),
// the 4 / CS groups of them different tokens.  With M the Pauli matrices of pauli_common.h, where reversion is
// the conjugate transpose, gx = M(gamma)^H M(dy) and the gradient of gamma is M(dy) M(xh)^H: 32 multiply-adds
// each, and <gx, x> is half the sum of the matrices' entries' products.  Every row is read once; the sums over
// the tokens stay in registers until the workgroup's last token, and are a plane of the workgroup's own then.
//
// Bound by memory: 32768 tokens of 256 multivectors with the residual's gradient, bf16, take 107 us in all, 102 of
// them here (537 MB: 5.2 TB/s, the rate of a copy of 1 GiB) and 4 in the planes' sum.  As two passes over the rows --
// dx, then gamma and beta -- the same took 291 us.  181 registers for four tokens at a time allow two workgroups on a
// CU; two tokens at a time and four workgroups took 4 us more, three workgroups with
// spilled registers 11 more.  Wider rows (d > 1024) would need more than four waves for a row; they take two passes,
// dx and then the parameters: 4096 tokens of 2048 multivectors with the residual's gradient, bf16, 195 us, where rows of
// 1024 take 61.5 (268 MB, 4.4 TB/s) and the 537 MB of one pass would take 106 at a copy's rate.
constexpr int kNbFusedMaxD = 1024, kNbMaxPlanes = 512;  // planes: two workgroups on each of 256 CUs

template <typename XT, typename GT, int CS, int NQ, int U>
__global__ __launch_bounds__(256) void norm_backward_kernel(const GT* __restrict__ dy, const XT* __restrict__ x, int N,
                                                            int d, const float* __restrict__ gamma, float two_eps,
                                                            const XT* residual, XT* dx, float* __restrict__ part) {
  constexpr int TS = 4 / CS;
  __shared__ float red[2][4][2 * U];  // [parity][wave][token of the batch: |x|^2, <gx, x>]
  __shared__ float4 sums[TS > 1 ? TS - 1 : 1][64 * CS][4];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int cw = wave % CS, tw = wave / CS;
  int col[NQ];
  bool live[NQ];
  float ga[NQ][2][4];  // the columns of gamma's matrix: (re, im) of entries 0 and 1
  float sg[NQ][8], sb[NQ][8];
#pragma unroll
  for (int q = 0; q < NQ; ++q) {
    const int i = (q * CS + cw) * 64 + lane;
    live[q] = i < d;
    col[q] = live[q] ? i : 0;
    float v[8];
    load_mv(gamma, col[q], v);
    blade_to_pauli(v, ga[q][0], ga[q][1]);
#pragma unroll
    for (int c = 0; c < 8; ++c) sg[q][c] = sb[q][c] = 0.f;
  }
  int parity = 0;
  for (int t0 = (blockIdx.x * TS + tw) * U, round = 0; round * gridDim.x * TS * U < N; ++round, t0 += gridDim.x * TS * U) {
    // (a token past the last repeats it, adds nothing and is not stored)
    RawMv<XT> rx[U][NQ], rr[U][NQ];
    RawMv<GT> rg[U][NQ];
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int q = 0; q < NQ; ++q) {
        const size_t n = (size_t)min(t0 + u, N - 1) * d + col[q];
        rx[u][q] = load_raw(x, n);
        rg[u][q] = load_raw(dy, n);
      }
    if (residual != nullptr) {
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int q = 0; q < NQ; ++q) rr[u][q] = load_raw(residual, (size_t)min(t0 + u, N - 1) * d + col[q]);
    }
    float gx[U][NQ][2][4], own[2 * U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float n2 = 0.f, dot = 0.f;
#pragma unroll
      for (int q = 0; q < NQ; ++q) {
        float v[8], xp[2][4], gp[2][4];
        unpack(rx[u][q], v);
        if (!live[q])
#pragma unroll
          for (int c = 0; c < 8; ++c) v[c] = 0.f;
#pragma unroll
        for (int c = 0; c < 8; ++c) n2 = __builtin_fmaf(v[c], v[c], n2);
        blade_to_pauli(v, xp[0], xp[1]);
        unpack(rg[u][q], v);
        if (!live[q])
#pragma unroll
          for (int c = 0; c < 8; ++c) v[c] = 0.f;
        blade_to_pauli(v, gp[0], gp[1]);
        // gx[r][b] = sum_a conj(gamma[a][r]) dy[a][b]
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const float* h = ga[q][r];
            const float* y = gp[b];
            const float re = __builtin_fmaf(h[3], y[3], __builtin_fmaf(h[2], y[2], __builtin_fmaf(h[1], y[1], h[0] * y[0])));
            const float im = __builtin_fmaf(-h[3], y[2], __builtin_fmaf(h[2], y[3], __builtin_fmaf(-h[1], y[0], h[0] * y[1])));
            gx[u][q][b][2 * r] = re;
            gx[u][q][b][2 * r + 1] = im;
            dot = __builtin_fmaf(re, xp[b][2 * r], __builtin_fmaf(im, xp[b][2 * r + 1], dot));
          }
      }
      own[2 * u] = n2;
      own[2 * u + 1] = dot;
    }
    const float s = wave_sums<2 * U>(own, lane);
    if ((lane & (64 / (2 * U) - 1)) == 0) red[parity][wave][wave_sums_of<2 * U>(lane)] = s;
    __syncthreads();
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float n2 = 0.f, dot = 0.f;
#pragma unroll
      for (int w = 0; w < CS; ++w) {
        n2 += red[parity][tw * CS + w][2 * u];
        dot += red[parity][tw * CS + w][2 * u + 1];
      }
      if (t0 + u >= N) continue;
      const float r = 1.0f / sqrtf(n2 / (float)d + two_eps);
      const float hr = 0.5f * r, w = -hr * (0.5f * dot) * r * r / (float)d;  // dx = (gx - x <gx, x> / (rms^2 d)) / rms
#pragma unroll
      for (int q = 0; q < NQ; ++q) {
        float v[8], g[8], xp[2][4], gp[2][4], o[8], e[8];
        unpack(rx[u][q], v);
        unpack(rg[u][q], g);
        blade_to_pauli(v, xp[0], xp[1]);
        blade_to_pauli(g, gp[0], gp[1]);
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
          for (int c = 0; c < 4; ++c) e[4 * b + c] = __builtin_fmaf(hr, gx[u][q][b][c], w * xp[b][c]);
        pauli_to_blade(e[0], e[1], e[4], e[5], e[2], e[3], e[6], e[7], o);
        if (residual != nullptr) {
          float f[8];
          unpack(rr[u][q], f);
#pragma unroll
          for (int c = 0; c < 8; ++c) o[c] += f[c];
        }
        if (live[q]) {
          store_mv(dx, (size_t)(t0 + u) * d + col[q], o);
#pragma unroll
          for (int c = 0; c < 8; ++c) sb[q][c] += g[c];
        }
        // M(dy) M(xh)^H, entry (a, c) = sum_b dy[a][b] conj(xh[c][b])
#pragma unroll
        for (int b = 0; b < 2; ++b) {
#pragma unroll
          for (int c = 0; c < 4; ++c) xp[b][c] *= r;
#pragma unroll
          for (int a = 0; a < 2; ++a)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              const float yr = gp[b][2 * a], yi = gp[b][2 * a + 1], xr = xp[b][2 * c], xi = xp[b][2 * c + 1];
              float* to = sg[q] + 4 * a + 2 * c;
              to[0] = __builtin_fmaf(yi, xi, __builtin_fmaf(yr, xr, to[0]));
              to[1] = __builtin_fmaf(-yr, xi, __builtin_fmaf(yi, xr, to[1]));
            }
        }
      }
    }
    parity ^= 1;  // the sums just read are written again after the next barrier
  }
  // the token groups' sums added in order
#pragma unroll
  for (int q = 0; q < NQ; ++q) {
    float o[16];
    pauli_to_blade(sg[q][0], sg[q][1], sg[q][2], sg[q][3], sg[q][4], sg[q][5], sg[q][6], sg[q][7], o);
#pragma unroll
    for (int c = 0; c < 8; ++c) {
      o[c] *= 0.5f;
      o[8 + c] = sb[q][c];
    }
    if constexpr (TS > 1) {
      __syncthreads();
      if (tw > 0)
#pragma unroll
        for (int c = 0; c < 4; ++c)
          sums[tw - 1][cw * 64 + lane][c] = make_float4(o[4 * c], o[4 * c + 1], o[4 * c + 2], o[4 * c + 3]);
      __syncthreads();
      if (tw == 0)
#pragma unroll
        for (int k = 0; k < TS - 1; ++k)
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const float4 m = sums[k][cw * 64 + lane][c];
            o[4 * c] += m.x; o[4 * c + 1] += m.y; o[4 * c + 2] += m.z; o[4 * c + 3] += m.w;
          }
    }
    if (tw == 0 && live[q]) {
      float* to = part + ((size_t)blockIdx.x * d + col[q]) * 16;
      store_mv(to, 0, o);
      store_mv(to, 1, o + 8);
    }
  }
}

// ---- few rows: one launch -------------------------------------------------------------------------
// The first workgroups take 16 multivectors each of gamma and beta, over all tokens: their waves find every token's
// rms, a row at a time, and then a thread adds every 64th token of its multivector; the sums meet by exchanges and in
// LDS, in an order that the sizes fix.  The other workgroups write dx, a wave a token.
//
// A second launch and a workspace are most of what a small call takes: 256 tokens of 64 multivectors, fp32, 10.5 us a
// call here, 15.2 with planes; 384 tokens 13.3 and 15.3, 512 tokens 15.6 and 15.2; 64 tokens of 512 multivectors,
// fp32, 19.5 and 15.
constexpr int kNbSmallTokens = 384, kNbSmallD = 256;
constexpr int kNbSmallUnits = 512;  // tokens times wave loads a row: the most that the first workgroups read through
constexpr int kNbCols = 16;

template <typename XT, typename GT>
__global__ __launch_bounds__(1024) void norm_backward_small_kernel(const GT* __restrict__ dy, const XT* __restrict__ x,
                                                                   int N, int d, const float* __restrict__ gamma,
                                                                   float two_eps, const XT* residual, XT* dx,
                                                                   float* __restrict__ dgamma, float* __restrict__ dbeta) {
  constexpr int U = 8;  // rows' pieces that a wave asks for together
  __shared__ float s_r[kNbSmallTokens];
  __shared__ float s_sum[16][16][kNbCols + 1];  // [wave][value][column]
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int blocks = (d + kNbCols - 1) / kNbCols;
  if ((int)blockIdx.x >= blocks) {
    const int t = ((int)blockIdx.x - blocks) * 16 + wave;
    if (t < N) norm_dx_row(dy, x, (size_t)t * d, d, gamma, two_eps, residual, dx, lane);
    return;
  }
  const int col = blockIdx.x * kNbCols + (lane & 15), slot = wave * 4 + (lane >> 4);  // of 64 slots for tokens
  for (int t0 = wave; t0 < N; t0 += 16 * U) {
    float n2[U];
#pragma unroll
    for (int u = 0; u < U; ++u) n2[u] = 0.f;
    for (int i = lane; i < d; i += 64) {
      RawMv<XT> m[U];
#pragma unroll
      for (int u = 0; u < U; ++u) m[u] = load_raw(x, (size_t)min(t0 + 16 * u, N - 1) * d + i);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        float v[8];
        unpack(m[u], v);
#pragma unroll
        for (int c = 0; c < 8; ++c) n2[u] = __builtin_fmaf(v[c], v[c], n2[u]);
      }
    }
    const float s = wave_sums<U>(n2, lane);
    const int t = t0 + 16 * wave_sums_of<U>(lane);
    if ((lane & (64 / U - 1)) == 0 && t < N) s_r[t] = 1.0f / sqrtf(s / (float)d + two_eps);
  }
  __syncthreads();
  float o[16];
#pragma unroll
  for (int c = 0; c < 16; ++c) o[c] = 0.f;
  if (col < d)
    for (int t0 = slot; t0 < N; t0 += 64 * 2) {
      RawMv<XT> mx[2];
      RawMv<GT> mg[2];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const size_t n = (size_t)min(t0 + 64 * u, N - 1) * d + col;
        mx[u] = load_raw(x, n);
        mg[u] = load_raw(dy, n);
      }
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        if (t0 + 64 * u >= N) break;
        float v[8], g[8], p[8];
        unpack(mx[u], v);
        unpack(mg[u], g);
        const float r = s_r[t0 + 64 * u];
#pragma unroll
        for (int c = 0; c < 8; ++c) v[c] *= r;
        product<false, true>(g, v, p);
#pragma unroll
        for (int c = 0; c < 8; ++c) {
          o[c] += p[c];
          o[8 + c] += g[c];
        }
      }
    }
#pragma unroll
  for (int c = 0; c < 16; ++c) {
    o[c] += __shfl_xor(o[c], 16);
    o[c] += __shfl_xor(o[c], 32);
    if (lane < 16) s_sum[wave][c][lane] = o[c];
  }
  __syncthreads();
  if (threadIdx.x < 16 * kNbCols) {
    const int c = threadIdx.x & 15, k = threadIdx.x >> 4, i = blockIdx.x * kNbCols + k;
    float s = 0.f;
#pragma unroll
    for (int w = 0; w < 16; ++w) s += s_sum[w][c][k];
    if (i < d && c < 8) dgamma[(size_t)i * 8 + c] = s;
    if (i < d && c >= 8) dbeta[(size_t)i * 8 + c - 8] = s;
  }
}

__global__ __launch_bounds__(1024) void norm_param_reduce_kernel(const float* __restrict__ part, int planes, int d,
                                                                 float* __restrict__ dgamma, float* __restrict__ dbeta) {
  add_planes(part, planes, d * 16, [&](int n, float v) {
    const size_t at = (size_t)(n >> 4) * 8 + (n & 7);
    if ((n & 15) < 8) dgamma[at] = v;  // (a choice between the two pointers would put them into scratch memory)
    else dbeta[at] = v;
  });
}

bool few_rows(int N, int d) {
  return d <= kNbSmallD && N <= kNbSmallTokens && (long long)N * ((d + 63) / 64) <= kNbSmallUnits;
}

// The tokens of a workgroup's batch and the planes of the one-pass kernel
int fused_batch(int d) { return d <= 64 ? 16 : d <= 128 ? 8 : d <= 256 ? 4 : d <= 512 ? 2 : 1; }
int planes_of(int N, int d) {
  if (d > kNbFusedMaxD) return (N + kNbPlaneTokens - 1) / kNbPlaneTokens;
  return std::min((N + fused_batch(d) - 1) / fused_batch(d), kNbMaxPlanes);
}
size_t rrms_bytes(int N, int d) { return d <= kNbFusedMaxD ? 0 : ((size_t)N * 4 + 255) / 256 * 256; }

template <typename XT, typename GT>
int launch(const void* dy, const void* x, int N, int d, const float* gamma, float two_eps, const void* residual,
           void* dx, float* dgamma, float* dbeta, void* workspace, hipStream_t stream) {
  if (few_rows(N, d)) {
    hipLaunchKernelGGL((norm_backward_small_kernel<XT, GT>), dim3((d + kNbCols - 1) / kNbCols + (N + 15) / 16), dim3(1024), 0,
                       stream, static_cast<const GT*>(dy), static_cast<const XT*>(x), N, d, gamma, two_eps,
                       static_cast<const XT*>(residual), static_cast<XT*>(dx), dgamma, dbeta);
    return check_launch("norm backward (few rows)");
  }
  float* rrms = static_cast<float*>(workspace);
  float* part = reinterpret_cast<float*>(static_cast<char*>(workspace) + rrms_bytes(N, d));
  const int planes = planes_of(N, d);
  if (N > 0 && d <= kNbFusedMaxD) {
#define YGG_NB(CS, NQ, U)                                                                                              \
  hipLaunchKernelGGL((norm_backward_kernel<XT, GT, CS, NQ, U>), dim3(planes), dim3(256), 0, stream,                    \
                     static_cast<const GT*>(dy), static_cast<const XT*>(x), N, d, gamma, two_eps,                      \
                     static_cast<const XT*>(residual), static_cast<XT*>(dx), part)
    if (d <= 64) YGG_NB(1, 1, 4);
    else if (d <= 128) YGG_NB(2, 1, 4);
    else if (d <= 256) YGG_NB(4, 1, 4);
    else if (d <= 512) YGG_NB(4, 2, 2);
    else YGG_NB(4, 4, 1);
#undef YGG_NB
    if (check_launch("norm backward")) return -1;
  } else if (N > 0) {
    hipLaunchKernelGGL((norm_dx_kernel<XT, GT>), dim3((N + 3) / 4), dim3(256), 0, stream, static_cast<const GT*>(dy),
                       static_cast<const XT*>(x), N, d, gamma, two_eps, static_cast<const XT*>(residual),
                       static_cast<XT*>(dx), rrms);
    if (check_launch("norm backward")) return -1;
    hipLaunchKernelGGL((norm_param_kernel<XT, GT>), dim3(planes, (d + 63) / 64), dim3(64), 0, stream,
                       static_cast<const GT*>(dy), static_cast<const XT*>(x), N, d, rrms, part);
    if (check_launch("norm backward (gamma and beta)")) return -1;
  }
  hipLaunchKernelGGL(norm_param_reduce_kernel, dim3((d * 16 + 31) / 32), dim3(1024), 0, stream, part, planes, d, dgamma,
                     dbeta);
  return check_launch("norm backward (reduction)");
}

}  // namespace
}  // namespace ygg

using namespace ygg;

YGG_API size_t ygg_clifford_layer_norm_backward_workspace_bytes(int N, int d) {
  if (N < 0 || d < 1 || d > kNbMaxD || few_rows(N, d)) return 0;
  return rrms_bytes(N, d) + (size_t)planes_of(N, d) * d * 16 * sizeof(float);
}

YGG_API int ygg_clifford_layer_norm_backward(const void* dy, int dy_dtype, const void* x, int x_dtype, int N, int d,
                                             const float* gamma, double eps, const void* residual_grad, void* dx,
                                             float* dgamma, float* dbeta, void* workspace, size_t workspace_bytes,
                                             hipStream_t stream) {
  YGG_CHECK_ARG(x_dtype == kF32 || x_dtype == kBF16, "ygg_clifford_layer_norm_backward: x dtype %d unsupported", x_dtype);
  YGG_CHECK_ARG(dy_dtype == kF32 || dy_dtype == kBF16, "ygg_clifford_layer_norm_backward: dy dtype %d unsupported",
                dy_dtype);
  YGG_CHECK_ARG(N >= 0 && N <= kNbMaxN && d >= 1 && d <= kNbMaxD,
                "ygg_clifford_layer_norm_backward: bad sizes N=%d d=%d (N <= %d, d <= %d)", N, d, kNbMaxN, kNbMaxD);
  YGG_CHECK_ARG(eps >= 0.0, "ygg_clifford_layer_norm_backward: eps must be non-negative");
  YGG_CHECK_ARG(gamma && dgamma && dbeta && (N == 0 || (dy && x && dx)),
                "ygg_clifford_layer_norm_backward: null pointer argument");
  const size_t need = ygg_clifford_layer_norm_backward_workspace_bytes(N, d);
  YGG_CHECK_ARG(need == 0 || (workspace && workspace_bytes >= need),
                "ygg_clifford_layer_norm_backward: workspace of %zu bytes, need %zu", workspace ? workspace_bytes : 0,
                need);
  const size_t mv = (size_t)N * d * 8, bx = mv * dtype_size(x_dtype), bp = (size_t)d * 8 * sizeof(float);
  YGG_CHECK_ARG(!overlap(dx, bx, dy, mv * dtype_size(dy_dtype)),
                "ygg_clifford_layer_norm_backward: dx is dy, or shares memory with it: other workgroups read dy");
  YGG_CHECK_ARG(!overlap(dx, bx, x, bx),
                "ygg_clifford_layer_norm_backward: dx is x, or shares memory with it: other workgroups read x");
  YGG_CHECK_ARG(dx == residual_grad || !overlap(dx, bx, residual_grad, bx),
                "ygg_clifford_layer_norm_backward: dx shares a part of residual_grad's memory");
  YGG_CHECK_ARG(!overlap(dgamma, bp, gamma, bp) && !overlap(dbeta, bp, gamma, bp),
                "ygg_clifford_layer_norm_backward: dgamma or dbeta shares memory with gamma, which other workgroups read");
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
