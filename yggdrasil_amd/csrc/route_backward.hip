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

#include <algorithm>
#include <type_traits>

#include "rows.h"
#include "ygg_common.h"

namespace ygg {
namespace {

constexpr int kRbMaxExperts = 64, kRbMaxK = 8;

// A token's weights, their gradients and experts (slots past k repeat the last: loads without conditions, which do
// not wait for one another), and dl of its slots.  All lanes that call it with the same t get the same values.
struct Slots {
  float w[kRbMaxK], g[kRbMaxK];
  int e[kRbMaxK];
};
__device__ __forceinline__ Slots load_slots(const int32_t* __restrict__ idx, const float* __restrict__ w,
                                            const float* __restrict__ g, size_t t, int k) {
  Slots o;
#pragma unroll
  for (int s = 0; s < kRbMaxK; ++s) {
    const size_t n = t * k + min(s, k - 1);
    o.w[s] = w[n];
    o.g[s] = g[n];
    o.e[s] = idx[n];
  }
  return o;
}
__device__ __forceinline__ void slot_gradients(const Slots& o, int k, float* dl) {
  float dot = 0.f;
#pragma unroll
  for (int s = 0; s < kRbMaxK; ++s)
    if (s < k) dot = __builtin_fmaf(o.w[s], o.g[s], dot);
#pragma unroll
  for (int s = 0; s < kRbMaxK; ++s) dl[s] = s < k && k > 1 ? o.w[s] * (o.g[s] - dot) : 0.f;
}

// A thread per (token, expert): every logit's gradient written once.
__global__ __launch_bounds__(256) void route_backward_kernel(const int32_t* __restrict__ idx, const float* __restrict__ w,
                                                             const float* __restrict__ g, int N, int E, int k,
                                                             float* __restrict__ dlogits) {
  for (size_t n = (size_t)blockIdx.x * 256 + threadIdx.x; n < (size_t)N * E; n += (size_t)gridDim.x * 256) {
    const size_t t = n / E;
    const int e = (int)(n - t * E);
    float dl[kRbMaxK], v = 0.f;
    const Slots o = load_slots(idx, w, g, t, k);
    slot_gradients(o, k, dl);
#pragma unroll
    for (int s = 0; s < kRbMaxK; ++s)
      if (s < k && o.e[s] == e) v += dl[s];
    dlogits[n] = v;
  }
}

__device__ __forceinline__ void add_energies(const float v[8], float en[4]) {
  en[0] = __builtin_fmaf(v[0], v[0], en[0]);
  en[3] = __builtin_fmaf(v[7], v[7], en[3]);
#pragma unroll
  for (int c = 0; c < 3; ++c) {
    en[1] = __builtin_fmaf(v[1 + c], v[1 + c], en[1]);
    en[2] = __builtin_fmaf(v[4 + c], v[4 + c], en[2]);
  }
}

// One token by a wave (a row of up to 64 NQ multivectors in registers, the rest read again from L2): its energies and
// dx (plus add).  slot(s, dl, e) gets the gradient of slot s, share(sh) the four shares, the same in every lane.
template <typename T, int NQ, class Slot, class Share>
__device__ __forceinline__ void energy_token(const T* x, int d, const float* W, int E, int k, const int32_t* idx,
                                             const float* w, const float* g, const T* add, T* dx, size_t t, int lane,
                                             Slot&& slot, Share&& share) {
  const size_t row = t * d;
  RawMv<T> rx[NQ], ra[NQ];
  // (lanes past the row load its last multivector again: under a condition the loads waited for one another)
#pragma unroll
  for (int q = 0; q < NQ; ++q) rx[q] = load_raw(x, row + min(lane + 64 * q, d - 1));
  if (add != nullptr) {
#pragma unroll
    for (int q = 0; q < NQ; ++q) ra[q] = load_raw(add, row + min(lane + 64 * q, d - 1));
  }
  // the slots' gradients and those of the shares (the same in every lane)
  float dl[kRbMaxK], ds[4] = {0.f, 0.f, 0.f, 0.f};
  const Slots o = load_slots(idx, w, g, t, k);
  slot_gradients(o, k, dl);
#pragma unroll
  for (int s = 0; s < kRbMaxK; ++s)
    if (s < k) {
      const int e = o.e[s];
      const bool known = e >= 0 && e < E;
      if (known)
#pragma unroll
        for (int h = 0; h < 4; ++h) ds[h] = __builtin_fmaf(dl[s], W[e * 4 + h], ds[h]);
      slot(s, dl[s], e);
    }
  float en[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int q = 0; q < NQ; ++q)
    if (lane + 64 * q < d) {
      float v[8];
      unpack(rx[q], v);
      add_energies(v, en);
    }
  for (int i = lane + 64 * NQ; i < d; i += 64) {
    float v[8];
    load_mv(x, row + i, v);
    add_energies(v, en);
  }
  const float sum = wave_sums<4>(en, lane);
  float sh[4], dot = 0.f;
#pragma unroll
  for (int h = 0; h < 4; ++h) en[h] = __shfl(sum, 16 * h);
  const float total = ((en[0] + en[1]) + (en[2] + en[3])) + 1e-12f;
#pragma unroll
  for (int h = 0; h < 4; ++h) {
    sh[h] = en[h] / total;
    dot = __builtin_fmaf(ds[h], sh[h], dot);
  }
  share(sh);
  float de[4];
#pragma unroll
  for (int h = 0; h < 4; ++h) de[h] = 2.f * (ds[h] - dot) / total;
  auto out = [&](float v[8], float o[8], int i) __attribute__((always_inline)) {
#pragma unroll
    for (int c = 0; c < 8; ++c) o[c] = __builtin_fmaf(v[c], de[c == 0 ? 0 : c < 4 ? 1 : c < 7 ? 2 : 3], o[c]);
    store_mv(dx, row + i, o);
  };
#pragma unroll
  for (int q = 0; q < NQ; ++q)
    if (lane + 64 * q < d) {
      float v[8], o[8] = {};
      unpack(rx[q], v);
      if (add != nullptr) unpack(ra[q], o);
      out(v, o, lane + 64 * q);
    }
  for (int i = lane + 64 * NQ; i < d; i += 64) {
    float v[8], o[8] = {};
    load_mv(x, row + i, v);
    if (add != nullptr) load_mv(add, row + i, o);
    out(v, o, i);
  }
}

// What lane e's expert has of a token's slots: its share of every grade and of the bias
__device__ __forceinline__ void add_slots(float4 share, const float* dl, const int* idx, int k, int lane, float s5[5]) {
  for (int s = 0; s < k; ++s) {
    const float v = idx[s] == lane ? dl[s] : 0.f;
    s5[0] = __builtin_fmaf(v, share.x, s5[0]);
    s5[1] = __builtin_fmaf(v, share.y, s5[1]);
    s5[2] = __builtin_fmaf(v, share.z, s5[2]);
    s5[3] = __builtin_fmaf(v, share.w, s5[3]);
    s5[4] += v;
  }
}

// A workgroup takes batches of up to 16 tokens, a wave one token at a time; for the parameters the tokens' shares
// and slot gradients stay in LDS.  Then lane e of every wave adds what expert e has of the wave's share of
// the slots.  The waves' sums are added in order at the end, and are a plane of the workgroup's own.
//
// Bound by memory: 32768 tokens of 256 multivectors, bf16, E = 64, k = 2 take 60 us in all, 49 of them here (268 MB
// read and written: 5.4 TB/s; a copy of 1 GiB runs at 5.1) and 5 in the planes' sum.  As three passes -- dx, then one
// workgroup per expert over all tokens -- the same took 244 us.
constexpr int kRbTokens = 16, kRbMaxPlanes = 2048;  // planes: eight workgroups on each of 256 CUs

template <typename T, int NQ>
__global__ __launch_bounds__(256) void energy_backward_kernel(const T* __restrict__ x, int N, int d,
                                                              const float* __restrict__ W, int E, int k,
                                                              const int32_t* __restrict__ idx,
                                                              const float* __restrict__ w, const float* __restrict__ g,
                                                              const T* add, T* dx, int tokens_per,
                                                              float* __restrict__ part) {
  __shared__ float4 s_share[kRbTokens];
  __shared__ float s_dl[kRbTokens * kRbMaxK];
  __shared__ int s_idx[kRbTokens * kRbMaxK];
  __shared__ float s_red[4][5][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  float s5[5] = {0.f, 0.f, 0.f, 0.f, 0.f};
  for (long long t0 = (long long)blockIdx.x * tokens_per; t0 < N; t0 += (long long)gridDim.x * tokens_per) {
    const int tokens = (int)min((long long)tokens_per, N - t0);
    for (int u = wave; u < tokens; u += 4) {
      const size_t t = (size_t)t0 + u;
      energy_token<T, NQ>(
          x, d, W, E, k, idx, w, g, add, dx, t, lane,
          [&](int s, float dl, int e) {
            if (lane == 0) {
              s_dl[u * kRbMaxK + s] = dl;
              s_idx[u * kRbMaxK + s] = e;
            }
          },
          [&](const float sh[4]) {
            if (lane == 0) s_share[u] = make_float4(sh[0], sh[1], sh[2], sh[3]);
          });
    }
    __syncthreads();
    for (int u = wave; u < tokens; u += 4) {
      add_slots(s_share[u], s_dl + u * kRbMaxK, s_idx + u * kRbMaxK, k, lane, s5);
    }
    __syncthreads();  // the next batch's slots
  }
#pragma unroll
  for (int h = 0; h < 5; ++h) s_red[wave][h][lane] = s5[h];
  __syncthreads();
  for (int i = threadIdx.x; i < 5 * E; i += 256) {  // plane: [5][E], the last row the bias
    const int h = i / E, e = i - h * E;
    part[(size_t)blockIdx.x * 5 * E + i] = (s_red[0][h][e] + s_red[1][h][e]) + (s_red[2][h][e] + s_red[3][h][e]);
  }
}

__global__ __launch_bounds__(1024) void router_param_kernel(const float* __restrict__ part, int planes, int E,
                                                            float* __restrict__ dW, float* __restrict__ db) {
  add_planes(part, planes, 5 * E, [&](int n, float v) {
    const int h = n / E, e = n - h * E;
    if (h < 4) dW[e * 4 + h] = v;
    else db[e] = v;
  });
}

// ---- few rows: one launch -------------------------------------------------------------------------
// The first workgroup sums the router's weight and bias over all tokens: every token's energies, a wave four rows at
// a time, then a thread a token for its slots, then lane e of a wave for what expert e has of its tokens, the waves'
// sums added in order.  The other workgroups write dx, a wave a token.
//
// A second launch and a workspace are most of what a small call takes: 256 tokens of 64 multivectors, fp32, 11.8 us a
// call here, 16.2 with planes; 384 tokens 15.1 and 16.4, 512 tokens 19.1 and 16.1; 32 tokens of 1024 multivectors,
// fp32, 18.1 and 16.4.
constexpr int kRbSmallTokens = 384, kRbSmallD = 512, kRbSmallSlots = 2048;
constexpr int kRbSmallUnits = 512;  // tokens times wave loads a row: the most that the first workgroup reads through

template <typename T, int NQ>
__global__ __launch_bounds__(1024) void energy_backward_small_kernel(
    const T* __restrict__ x, int N, int d, const float* __restrict__ W, int E, int k, const int32_t* __restrict__ idx,
    const float* __restrict__ w, const float* __restrict__ g, const T* add, T* dx, float* __restrict__ dW,
    float* __restrict__ db) {
  constexpr int U = 4;  // rows' pieces that a wave asks for together
  __shared__ float4 s_share[kRbSmallTokens];  // energies first
  __shared__ __attribute__((aligned(16))) float s_dl[kRbSmallTokens * kRbMaxK];
  __shared__ __attribute__((aligned(16))) int s_idx[kRbSmallTokens * kRbMaxK];
  __shared__ float s_red[16][5][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (blockIdx.x > 0) {
    const int t = ((int)blockIdx.x - 1) * 16 + wave;
    if (t < N) energy_token<T, NQ>(x, d, W, E, k, idx, w, g, add, dx, t, lane, [](int, float, int) {}, [](const float*) {});
    return;
  }
  Slots own;  // thread t's token t, asked for before the rows
  if ((int)threadIdx.x < N) own = load_slots(idx, w, g, threadIdx.x, k);
  for (int t0 = wave; t0 < N; t0 += 16 * U) {
    float en[4 * U];
#pragma unroll
    for (int n = 0; n < 4 * U; ++n) en[n] = 0.f;
    for (int i = lane; i < d; i += 64) {
      RawMv<T> m[U];
#pragma unroll
      for (int u = 0; u < U; ++u) m[u] = load_raw(x, (size_t)min(t0 + 16 * u, N - 1) * d + i);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        float v[8];
        unpack(m[u], v);
        add_energies(v, en + 4 * u);
      }
    }
    const float s = wave_sums<4 * U>(en, lane);
    const int n = wave_sums_of<4 * U>(lane), t = t0 + 16 * (n >> 2);
    if ((lane & (64 / (4 * U) - 1)) == 0 && t < N) reinterpret_cast<float*>(s_share + t)[n & 3] = s;
  }
  __syncthreads();
  if ((int)threadIdx.x < N) {
    const int t = threadIdx.x;
    float dl[kRbMaxK];
    slot_gradients(own, k, dl);
#pragma unroll
    for (int s = 0; s < kRbMaxK; ++s) {  // (slots past k: no expert)
      s_dl[t * kRbMaxK + s] = dl[s];
      s_idx[t * kRbMaxK + s] = s < k ? own.e[s] : -1;
    }
    const float4 e = s_share[t];
    const float total = ((e.x + e.y) + (e.z + e.w)) + 1e-12f;
    s_share[t] = make_float4(e.x / total, e.y / total, e.z / total, e.w / total);
  }
  __syncthreads();
  float s5[5] = {0.f, 0.f, 0.f, 0.f, 0.f};
  for (int t = wave; t < N; t += 16)
    for (int s = 0; s < k; s += 4) {
      const float4 share = s_share[t], dl = *reinterpret_cast<const float4*>(s_dl + t * kRbMaxK + s);
      const int4 at = *reinterpret_cast<const int4*>(s_idx + t * kRbMaxK + s);
      const float v = ((at.x == lane ? dl.x : 0.f) + (at.y == lane ? dl.y : 0.f)) +
                      ((at.z == lane ? dl.z : 0.f) + (at.w == lane ? dl.w : 0.f));
      s5[0] = __builtin_fmaf(v, share.x, s5[0]);
      s5[1] = __builtin_fmaf(v, share.y, s5[1]);
      s5[2] = __builtin_fmaf(v, share.z, s5[2]);
      s5[3] = __builtin_fmaf(v, share.w, s5[3]);
      s5[4] += v;
    }
#pragma unroll
  for (int h = 0; h < 5; ++h) s_red[wave][h][lane] = s5[h];
  __syncthreads();
  for (int i = threadIdx.x; i < 5 * E; i += 1024) {
    const int h = i / E, e = i - h * E;
    float s = 0.f;
#pragma unroll
    for (int q = 0; q < 16; ++q) s += s_red[q][h][e];
    if (h < 4) dW[e * 4 + h] = s;
    else db[e] = s;
  }
}

bool few_rows(int N, int d, int k) {
  return d <= kRbSmallD && N <= kRbSmallTokens && N * k <= kRbSmallSlots && (long long)N * ((d + 63) / 64) <= kRbSmallUnits;
}

// Tokens of a batch: enough workgroups to fill the chip first, then larger batches, then several a workgroup
int batch_tokens(int N) { return std::min(kRbTokens, std::max(4, (N / kRbMaxPlanes + 3) / 4 * 4)); }
int route_planes(int N) {
  const int per = batch_tokens(N);
  return std::min(kRbMaxPlanes, N / per + (N % per != 0));
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
  const size_t n = (size_t)N * E, slots = (size_t)N * k * 4;
  YGG_CHECK_ARG(!overlap(dlogits, n * 4, topk_idx, slots) && !overlap(dlogits, n * 4, topk_w, slots) &&
                    !overlap(dlogits, n * 4, dtopk_w, slots),
                "ygg_route_backward: dlogits shares memory with the routing, which other threads read");
  const unsigned groups = (unsigned)std::min<size_t>((n + 255) / 256, 1u << 23);  // a launch holds below 2^32 threads
  hipLaunchKernelGGL(route_backward_kernel, dim3(groups), dim3(256), 0, stream, topk_idx, topk_w, dtopk_w, N, E, k,
                     dlogits);
  return check_launch("ygg_route_backward");
}

YGG_API size_t ygg_route_energy_backward_workspace_bytes(int N, int d, int E, int k) {
  if (N < 0 || d < 1 || E < 1 || k < 1 || few_rows(N, d, k)) return 0;
  return (size_t)route_planes(N) * 5 * E * sizeof(float);
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
  const size_t need = ygg_route_energy_backward_workspace_bytes(N, d, E, k);
  YGG_CHECK_ARG(need == 0 || (workspace && workspace_bytes >= need),
                "ygg_route_energy_backward: workspace of %zu bytes, need %zu", workspace ? workspace_bytes : 0, need);
  const size_t bx = (size_t)N * d * 8 * dtype_size(x_dtype), bw = (size_t)E * 4 * sizeof(float);
  YGG_CHECK_ARG(!overlap(dx, bx, x, bx), "ygg_route_energy_backward: dx is x, or shares memory with it: other workgroups read x");
  YGG_CHECK_ARG(dx == dx_add || !overlap(dx, bx, dx_add, bx),
                "ygg_route_energy_backward: dx shares a part of dx_add's memory");
  YGG_CHECK_ARG(!overlap(drouter_w, bw, router_w, bw) && !overlap(drouter_b, bw / 4, router_w, bw),
                "ygg_route_energy_backward: a gradient shares memory with router_w, which other workgroups read");
  if (few_rows(N, d, k)) {
    auto run = [&](auto* xt, auto nq) {
      using T = std::remove_const_t<std::remove_pointer_t<decltype(xt)>>;
      hipLaunchKernelGGL((energy_backward_small_kernel<T, decltype(nq)::value>), dim3(1 + (N + 15) / 16), dim3(1024), 0, stream,
                         xt, N, d, router_w, E, k, topk_idx, topk_w, dtopk_w, static_cast<const T*>(dx_add),
                         static_cast<T*>(dx), drouter_w, drouter_b);
    };
    auto by_width = [&](auto* xt) {
      if (d <= 64) run(xt, std::integral_constant<int, 1>{});
      else run(xt, std::integral_constant<int, 2>{});
    };
    if (x_dtype == kF32) by_width(static_cast<const float*>(x));
    else by_width(static_cast<const uint16_t*>(x));
    return check_launch("ygg_route_energy_backward (few rows)");
  }
  float* part = static_cast<float*>(workspace);
  if (N > 0) {
    auto run = [&](auto* xt, auto nq) {
      using T = std::remove_const_t<std::remove_pointer_t<decltype(xt)>>;
      hipLaunchKernelGGL((energy_backward_kernel<T, decltype(nq)::value>), dim3(route_planes(N)), dim3(256), 0, stream, xt,
                         N, d, router_w, E, k, topk_idx, topk_w, dtopk_w, static_cast<const T*>(dx_add),
                         static_cast<T*>(dx), batch_tokens(N), part);
    };
    auto by_width = [&](auto* xt) {
      if (d <= 64) run(xt, std::integral_constant<int, 1>{});
      else if (d <= 128) run(xt, std::integral_constant<int, 2>{});
      else run(xt, std::integral_constant<int, 4>{});
    };
    if (x_dtype == kF32) by_width(static_cast<const float*>(x));
    else by_width(static_cast<const uint16_t*>(x));
    if (check_launch("ygg_route_energy_backward")) return -1;
  }
  hipLaunchKernelGGL(router_param_kernel, dim3((5 * E + 31) / 32), dim3(1024), 0, stream, part,
                     N > 0 ? route_planes(N) : 0, E, drouter_w, drouter_b);
  return check_launch("ygg_route_energy_backward (parameters)");
}
