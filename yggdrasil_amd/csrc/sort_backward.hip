// sort_backward.hip -- the gradients of the sort by expert and of the weighted way back (hlm_block.py:178, 180-181;
// forward: dispatch.hip; the reference has no MoE backward, hlm_block.py:202-206).
//
//   out_t = sum_s w_ts y[slot_ts]:   dy[slot_ts] = w_ts dout_t,   dw_ts = <dout_t, y[slot_ts]>
//   x_sorted[slot_ts] = x_t:         dx_t = sum_s dx_sorted[slot_ts]  (and what reaches x_t past the sort)
//
// Every row is read once and written once: both are bound by memory.  A slot names one row, so nothing is added
// across workgroups; a token's rows are added in slot order, in fp32.  A slot outside the rows is left out.

#include <hip/hip_runtime.h>

#include <algorithm>

#include "rows.h"
#include "ygg_common.h"

namespace ygg {
namespace {

constexpr int kMaxTopK = 8;

enum DyLayout : int { kDyBlade = 0, kDyPauli = 1 };

template <int LAYOUT>
__device__ __forceinline__ void store_dy(uint16_t* dy, size_t row, int i, int d, const float g[8], const float c[8], float w) {
  if constexpr (LAYOUT == kDyPauli) {  // half-rows (c: the Pauli columns of g)
    uint16_t* to = dy + (row * 2 * d + i) * 4;
    *reinterpret_cast<uint2*>(to) = make_uint2(pack2_bf16(w * c[0], w * c[1]), pack2_bf16(w * c[2], w * c[3]));
    *reinterpret_cast<uint2*>(to + (size_t)d * 4) = make_uint2(pack2_bf16(w * c[4], w * c[5]), pack2_bf16(w * c[6], w * c[7]));
  } else {
    float o[8];
#pragma unroll
    for (int q = 0; q < 8; ++q) o[q] = w * g[q];
    store_mv(dy, row * d + i, o);
  }
}
template <int LAYOUT>
__device__ __forceinline__ void store_dy(float* dy, size_t row, int i, int d, const float g[8], const float[8], float w) {
  float o[8];
#pragma unroll
  for (int q = 0; q < 8; ++q) o[q] = w * g[q];
  if constexpr (LAYOUT == kDyPauli) store_pauli_f32(dy + (row * d + i) * 8, o);
  else store_mv(dy, row * d + i, o);
}

// One wave per token (bf16 half-rows, 8192 tokens, d = 128, k = 4: 25.7 us, 151 MB at 5.9 TB/s).
template <typename TD, typename TY, int LAYOUT>
__global__ __launch_bounds__(256) void combine_backward_kernel(const TD* __restrict__ dout, const TY* __restrict__ y, int N,
                                                               int k, int d, int P, const float* __restrict__ topk_w,
                                                               const int32_t* __restrict__ slot_pos, TY* __restrict__ dy,
                                                               float* __restrict__ dtopk_w) {
  const int lane = threadIdx.x & 63;
  const int t = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (t >= N) return;
  float dot[kMaxTopK] = {};
  for (int i = lane; i < d; i += 64) {
    float g[8], c[8];
    load_mv(dout, (size_t)t * d + i, g);
    if constexpr (LAYOUT == kDyPauli && sizeof(TY) == 2) blade_to_pauli(g, c, c + 4);
#pragma unroll
    for (int s = 0; s < kMaxTopK; ++s) {
      if (s >= k) break;
      const int at = slot_pos[(size_t)t * k + s];
      if ((unsigned)at >= (unsigned)P) continue;
      const size_t row = (size_t)at;
      store_dy<LAYOUT>(dy, row, i, d, g, c, topk_w[(size_t)t * k + s]);
      if (dtopk_w != nullptr) {
        float v[8];
        load_mv(y, row * d + i, v);
#pragma unroll
        for (int q = 0; q < 8; ++q) dot[s] = __builtin_fmaf(g[q], v[q], dot[s]);
      }
    }
  }
  if (dtopk_w != nullptr) {
    const float sum = wave_sums<kMaxTopK>(dot, lane);
    const int s = wave_sums_of<kMaxTopK>(lane);
    if ((lane & (64 / kMaxTopK - 1)) == 0 && s < k) dtopk_w[(size_t)t * k + s] = sum;
  }
}

// A thread per multivector of a token (bf16, 8192 tokens, d = 128, k = 4: 17.6 us, 84 MB at 4.8 TB/s).
template <typename T>
__global__ __launch_bounds__(256) void dispatch_backward_kernel(const T* __restrict__ dxs, int k, int d, int P,
                                                                const int32_t* __restrict__ slot_pos,
                                                                const T* __restrict__ add, T* __restrict__ dx) {
  const int t = blockIdx.x;
  const int32_t* sp = slot_pos + (size_t)t * k;  // (the same for every thread: scalar loads)
  for (int i = threadIdx.x; i < d; i += blockDim.x) {
    float o[8] = {};
    if (add != nullptr) load_mv(add, (size_t)t * d + i, o);
    RawMv<T> r[kMaxTopK];
#pragma unroll
    for (int s = 0; s < kMaxTopK; ++s)
      if (s < k && (unsigned)sp[s] < (unsigned)P) r[s] = load_raw(dxs, (size_t)sp[s] * d + i);
#pragma unroll
    for (int s = 0; s < kMaxTopK; ++s)
      if (s < k && (unsigned)sp[s] < (unsigned)P) {
        float v[8];
        unpack(r[s], v);
#pragma unroll
        for (int c = 0; c < 8; ++c) o[c] += v[c];
      }
    store_mv(dx, (size_t)t * d + i, o);
  }
}

// tokens of a launch: a grid holds fewer than 2^32 threads
constexpr int kLaunchTokens = 1 << 22;

template <typename TD, typename TY>
int launch_combine(const void* dout, const void* y, int N, int k, int d, int P, const float* w, const int32_t* slots, void* dy,
                   int layout, float* dw, hipStream_t stream) {
  const TY* Y = static_cast<const TY*>(y);
  TY* O = static_cast<TY*>(dy);
  for (size_t t0 = 0; t0 < (size_t)N; t0 += kLaunchTokens) {
    const int n = (int)std::min<size_t>(N - t0, kLaunchTokens);
    const unsigned grid = (unsigned)(n + 3) / 4;
    const TD* const D = static_cast<const TD*>(dout) + t0 * d * 8;
    const float* const W = w + t0 * k;
    const int32_t* const S = slots + t0 * k;
    float* const DW = dw ? dw + t0 * k : nullptr;
    if (layout == kDyPauli) combine_backward_kernel<TD, TY, kDyPauli><<<grid, 256, 0, stream>>>(D, Y, n, k, d, P, W, S, O, DW);
    else combine_backward_kernel<TD, TY, kDyBlade><<<grid, 256, 0, stream>>>(D, Y, n, k, d, P, W, S, O, DW);
    if (check_launch("combine_backward")) return -1;
  }
  return 0;
}

// Workgroups no wider than the row's whole waves.
template <typename T>
int launch_dispatch(const void* dxs, int N, int k, int d, int P, const int32_t* slots, const void* add, void* dx,
                    hipStream_t stream) {
  const unsigned threads = d <= 64 ? 64 : d <= 128 ? 128 : 256;
  for (size_t t0 = 0; t0 < (size_t)N; t0 += kLaunchTokens) {
    const unsigned n = (unsigned)std::min<size_t>(N - t0, kLaunchTokens);
    const size_t at = t0 * d * 8;
    dispatch_backward_kernel<T><<<n, threads, 0, stream>>>(static_cast<const T*>(dxs), k, d, P, slots + t0 * k,
                                                           add ? static_cast<const T*>(add) + at : nullptr,
                                                           static_cast<T*>(dx) + at);
    if (check_launch("dispatch_backward")) return -1;
  }
  return 0;
}

}  // namespace

int combine_backward_bf16(const void* dout, const void* y, int N, int k, int d, const float* topk_w, const int32_t* slot_pos,
                          void* dy, float* dtopk_w, hipStream_t stream) {
  return launch_combine<uint16_t, uint16_t>(dout, y, N, k, d, N * k, topk_w, slot_pos, dy, kDyPauli, dtopk_w, stream);
}

int dispatch_backward_bf16(const void* dxs, int N, int k, int d, const int32_t* slot_pos, const void* add, void* dx,
                           hipStream_t stream) {
  return launch_dispatch<uint16_t>(dxs, N, k, d, N * k, slot_pos, add, dx, stream);
}

}  // namespace ygg

using namespace ygg;

YGG_API int ygg_combine_backward(const void* dout, int dout_dtype, const void* y_sorted, int N, int k, int d, int P,
                                 const float* topk_w, const int32_t* slot_pos, void* dy, int dy_dtype, int dy_layout,
                                 float* dtopk_w, hipStream_t stream) {
  YGG_CHECK_ARG(N >= 0 && d >= 1 && k >= 1 && k <= kMaxTopK && P >= 0, "ygg_combine_backward: bad sizes N=%d k=%d d=%d P=%d (k <= %d)",
                N, k, d, P, kMaxTopK);
  YGG_CHECK_ARG((dout_dtype == kF32 || dout_dtype == kBF16) && (dy_dtype == kF32 || dy_dtype == kBF16),
                "ygg_combine_backward: dtypes %d, %d unsupported", dout_dtype, dy_dtype);
  YGG_CHECK_ARG(dy_layout == kDyBlade || dy_layout == kDyPauli, "ygg_combine_backward: layout %d", dy_layout);
  if (N == 0) return 0;
  YGG_CHECK_ARG(dout && topk_w && slot_pos && (dy || P == 0), "ygg_combine_backward: null pointer");
  YGG_CHECK_ARG(!y_sorted == !dtopk_w || (P == 0 && dtopk_w), "ygg_combine_backward: the routing weights' gradient needs y_sorted, and y_sorted it");
  const size_t db = (size_t)N * d * 8 * dtype_size(dout_dtype), yb = (size_t)P * d * 8 * dtype_size(dy_dtype);
  const size_t slots = (size_t)N * k * 4;
  YGG_CHECK_ARG(!overlap(dy, yb, dout, db) && !overlap(dy, yb, y_sorted, yb) && !overlap(dy, yb, topk_w, slots) &&
                    !overlap(dy, yb, slot_pos, slots) && !overlap(dy, yb, dtopk_w, slots) && !overlap(dtopk_w, slots, dout, db) &&
                    !overlap(dtopk_w, slots, y_sorted, yb) && !overlap(dtopk_w, slots, topk_w, slots) &&
                    !overlap(dtopk_w, slots, slot_pos, slots),
                "ygg_combine_backward: outputs must not share memory with inputs or each other");
  if (dout_dtype == kF32)
    return dy_dtype == kF32
               ? launch_combine<float, float>(dout, y_sorted, N, k, d, P, topk_w, slot_pos, dy, dy_layout, dtopk_w, stream)
               : launch_combine<float, uint16_t>(dout, y_sorted, N, k, d, P, topk_w, slot_pos, dy, dy_layout, dtopk_w, stream);
  return dy_dtype == kF32
             ? launch_combine<uint16_t, float>(dout, y_sorted, N, k, d, P, topk_w, slot_pos, dy, dy_layout, dtopk_w, stream)
             : launch_combine<uint16_t, uint16_t>(dout, y_sorted, N, k, d, P, topk_w, slot_pos, dy, dy_layout, dtopk_w, stream);
}

YGG_API int ygg_dispatch_backward(const void* dx_sorted, int dtype, int N, int k, int d, int P, const int32_t* slot_pos,
                                  const void* dx_add, void* dx, hipStream_t stream) {
  YGG_CHECK_ARG(N >= 0 && d >= 1 && k >= 1 && k <= kMaxTopK && P >= 0, "ygg_dispatch_backward: bad sizes N=%d k=%d d=%d P=%d (k <= %d)",
                N, k, d, P, kMaxTopK);
  YGG_CHECK_ARG(dtype == kF32 || dtype == kBF16, "ygg_dispatch_backward: dtype %d unsupported", dtype);
  if (N == 0) return 0;
  YGG_CHECK_ARG((dx_sorted || P == 0) && slot_pos && dx, "ygg_dispatch_backward: null pointer");
  const size_t es = dtype_size(dtype), nb = (size_t)N * d * 8 * es, pb = (size_t)P * d * 8 * es;
  YGG_CHECK_ARG(!overlap(dx, nb, dx_sorted, pb) && !overlap(dx, nb, slot_pos, (size_t)N * k * 4) &&
                    (dx == dx_add || !overlap(dx, nb, dx_add, nb)),
                "ygg_dispatch_backward: dx must not share memory with dx_sorted, slot_pos or a part of dx_add");
  return (dtype == kF32 ? launch_dispatch<float> : launch_dispatch<uint16_t>)(dx_sorted, N, k, d, P, slot_pos, dx_add, dx, stream);
}
