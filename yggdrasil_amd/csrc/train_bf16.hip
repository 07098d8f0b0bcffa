// train_bf16.hip -- a training step of the bf16 layer: the forward that keeps what its backward reads, and the
// backward (the fp32 layer's: capi.hip, backward.hip; the reference has none, hlm_block.py:202-206).
//
// Forward (hlm_block.py:154-183): routing and x's Pauli half-rows, h = act(W_up x + b_up) with its rows before
// the activation kept, y = W_down h + b_down, out = sum of the slots' weighted rows.  Backward:
//   dy_r   = w_r dout_t                              (the combine's; dw_r = <dout_t, y_r>)
//   dh_r   = act'(h_pre_r) (~W_down dy_r)            (ygg_pauli_grouped_input_grad)
//   dx_t   = sum over the slots of ~W_up dh_r        (and dout_t, when the forward added x)
//   dW_down = sum dy_r ~h_r,  dW_up = sum dh_r ~x_t  (ygg_grouped_weight_grad_pauli_bf16)
// Rows between two operators are bf16, as the forward's are; every sum inside one is fp32.

#include <hip/hip_runtime.h>

#include <algorithm>

#include "rows.h"
#include "ygg_common.h"

extern "C" int ygg_combine(const void*, int, int, int, int, int, const int32_t*, const float*, const int32_t*,
                           const void*, void*, int, hipStream_t);
extern "C" int ygg_pauli_grouped_linear(const void*, int, int, const int32_t*, int, const void*, const float*,
                                        const int32_t*, int, int, int, int, void*, int, int, hipStream_t);
extern "C" int ygg_pauli_grouped_input_grad(const void*, int, const void*, const int32_t*, int, int, int, int, const void*,
                                            void*, int, int, hipStream_t);
extern "C" size_t ygg_route_workspace_bytes(int N, int E, int k);

namespace ygg {
namespace {

constexpr int kMaxTopK = 8;

// One wave per token: dy[slot] = w dout_t as Pauli half-rows and dtopk_w = <dout_t, y[slot]> (when y is not
// NULL).  Bound by memory: dout and y are read once, dy is written once (8192 tokens, d = 128, k = 4: 25.7 us, 151 MB
// at 5.9 TB/s).
__global__ __launch_bounds__(256) void combine_backward_bf16_kernel(const uint16_t* __restrict__ dout,
                                                                    const uint16_t* __restrict__ y, int N, int k, int d,
                                                                    const float* __restrict__ topk_w,
                                                                    const int32_t* __restrict__ slot_pos,
                                                                    uint16_t* __restrict__ dy, float* __restrict__ dtopk_w) {
  const int lane = threadIdx.x & 63;
  const int t = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (t >= N) return;
  float dot[kMaxTopK] = {};
  for (int i = lane; i < d; i += 64) {
    float g[8];
    load_mv(dout, (size_t)t * d + i, g);
    float c0[4], c1[4];
    blade_to_pauli(g, c0, c1);
#pragma unroll
    for (int s = 0; s < kMaxTopK; ++s) {
      if (s >= k) break;
      const size_t row = (size_t)slot_pos[(size_t)t * k + s];
      const float w = topk_w[(size_t)t * k + s];
      uint16_t* to = dy + (row * 2 * d + i) * 4;
      *reinterpret_cast<uint2*>(to) = make_uint2(pack2_bf16(w * c0[0], w * c0[1]), pack2_bf16(w * c0[2], w * c0[3]));
      *reinterpret_cast<uint2*>(to + (size_t)d * 4) =
          make_uint2(pack2_bf16(w * c1[0], w * c1[1]), pack2_bf16(w * c1[2], w * c1[3]));
      if (y != nullptr) {
        float v[8];
        load_mv(y, row * d + i, v);
#pragma unroll
        for (int c = 0; c < 8; ++c) dot[s] = __builtin_fmaf(g[c], v[c], dot[s]);
      }
    }
  }
  if (y != nullptr) {
    const float sum = wave_sums<kMaxTopK>(dot, lane);
    const int s = wave_sums_of<kMaxTopK>(lane);
    if ((lane & (64 / kMaxTopK - 1)) == 0 && s < k) dtopk_w[(size_t)t * k + s] = sum;
  }
}

// dx_t = (dout_t) + sum over the slots, in slot order, of dxs[slot_pos]; a thread per multivector.  Bound by memory: the
// rows read and dx written once (8192 tokens, d = 128, k = 4: 17.6 us, 84 MB at 4.8 TB/s).
__global__ __launch_bounds__(256) void dispatch_backward_bf16_kernel(const uint16_t* __restrict__ dxs, int N, int k, int d,
                                                                     const int32_t* __restrict__ slot_pos,
                                                                     const uint16_t* __restrict__ dout,
                                                                     uint16_t* __restrict__ dx) {
  const int t = blockIdx.x;
  const int32_t* sp = slot_pos + (size_t)t * k;  // (the same for every thread: scalar loads)
  for (int i = threadIdx.x; i < d; i += blockDim.x) {
    float o[8] = {};
    if (dout != nullptr) load_mv(dout, (size_t)t * d + i, o);
    RawMv<uint16_t> r[kMaxTopK];
#pragma unroll
    for (int s = 0; s < kMaxTopK; ++s)
      if (s < k) r[s] = load_raw(dxs, (size_t)sp[s] * d + i);
#pragma unroll
    for (int s = 0; s < kMaxTopK; ++s)
      if (s < k) {
        float v[8];
        unpack(r[s], v);
#pragma unroll
        for (int c = 0; c < 8; ++c) o[c] += v[c];
      }
    store_mv(dx, (size_t)t * d + i, o);
  }
}

size_t align256(size_t b) { return (b + 255) & ~(size_t)255; }

// What the forward keeps, each region on 256 bytes
struct Saved {
  size_t perm, slot_pos, x, h_pre, h, y, total;
};
Saved saved_of(int N, int d, int F, int k) {
  const size_t P = (size_t)N * k;
  Saved s;
  size_t at = 0;
  auto put = [&](size_t bytes) {
    const size_t o = at;
    at += align256(bytes);
    return o;
  };
  s.perm = put(P * 4);
  s.slot_pos = put(P * 4);
  s.x = put((size_t)N * d * 16);   // Pauli half-rows
  s.h_pre = put(P * F * 16);       // blade rows
  s.h = put(P * F * 16);           // Pauli half-rows
  s.y = put(P * d * 16);           // blade rows
  s.total = at;
  return s;
}

// nullptr, or why the sizes cannot be computed (the layer's own limits: capi.hip)
int check_sizes(const char* who, int N, int d, int F, int E, int k, int act) {
  YGG_CHECK_ARG(N >= 0 && d >= 2 && d % 2 == 0 && F >= 2 && F % 2 == 0 && E >= 1 && E <= 64 && k >= 1 && k <= kMaxTopK &&
                    k <= E, "%s: bad sizes N=%d d=%d F=%d E=%d k=%d (d and F even, E <= 64, k <= min(%d, E))", who, N, d, F,
                E, k, kMaxTopK);
  YGG_CHECK_ARG(act >= kActNone && act <= kActSigmoid, "%s: activation %d", who, act);
  YGG_CHECK_ARG((long long)N * k <= 0x7fffffffLL, "%s: N k = %lld token-expert rows exceed 2^31 - 1", who,
                (long long)N * k);
  if (N == 0) return 0;
  const int P = N * k;
  const char* why = pauli_size_limit(/*Pauli rows*/ 1, N, /*gathered*/ true, P, E, d, F, /*Pauli rows*/ 0, kBF16);
  if (!why) why = pauli_size_limit(1, P, false, P, E, F, d, /*blade*/ 1, kBF16);
  if (!why) why = pauli_size_limit(1, P, false, P, E, d, F, /*Pauli rows*/ 0, kBF16);
  if (!why) why = weight_grad_bf16_limit(P, E, d, F, /*gathered*/ true, N);
  if (!why) why = weight_grad_bf16_limit(P, E, F, d, false, P);
  YGG_CHECK_ARG(!why, "%s: %s (N=%d d=%d F=%d E=%d k=%d)", who, why, N, d, F, E, k);
  return 0;
}

}  // namespace
}  // namespace ygg

using namespace ygg;

YGG_API size_t ygg_moe_train_bf16_saved_bytes(int N, int d, int F, int E, int k) {
  if (N < 0 || d < 1 || F < 1 || E < 1 || k < 1) return 0;
  return saved_of(N, d, F, k).total;
}

YGG_API size_t ygg_moe_forward_train_bf16_workspace_bytes(int N, int d, int F, int E, int k) {
  if (N < 0 || d < 1 || F < 1 || E < 1 || k < 1) return 0;
  return align256((size_t)N * E * 4) + align256(ygg_route_workspace_bytes(N, E, k));
}

YGG_API int ygg_moe_forward_train_bf16(const void* x, int N, int d, int F, int E, int k, int act, const float* logits,
                                       const float* router_w, const float* router_b, const void* w_up, const float* b_up,
                                       const void* w_down, const float* b_down, const void* residual, void* out,
                                       int32_t* topk_idx, float* topk_w, int32_t* counts, int32_t* offsets, void* saved,
                                       size_t saved_bytes, void* workspace, size_t workspace_bytes, hipStream_t stream) {
  if (check_sizes("ygg_moe_forward_train_bf16", N, d, F, E, k, act)) return -1;
  YGG_CHECK_ARG(counts && offsets, "ygg_moe_forward_train_bf16: null pointer");
  YGG_CHECK_ARG(N == 0 || (x && w_up && w_down && out && topk_idx && topk_w && saved && workspace),
                "ygg_moe_forward_train_bf16: null pointer");
  YGG_CHECK_ARG(N == 0 || logits || (router_w && router_b), "ygg_moe_forward_train_bf16: need logits or router parameters");
  const Saved at = saved_of(N, d, F, k);
  YGG_CHECK_ARG(saved_bytes >= at.total, "ygg_moe_forward_train_bf16: %zu bytes to keep rows in, need %zu", saved_bytes,
                at.total);
  const size_t need = ygg_moe_forward_train_bf16_workspace_bytes(N, d, F, E, k);
  YGG_CHECK_ARG(workspace_bytes >= need, "ygg_moe_forward_train_bf16: workspace of %zu bytes, need %zu", workspace_bytes,
                need);
  char* const keep = static_cast<char*>(saved);
  RowConvert none;
  if (N == 0)
    return route_convert(nullptr, 0, E, k, nullptr, nullptr, counts, offsets, nullptr, nullptr, nullptr, 0, none, stream);
  const int P = N * k;
  int32_t* perm = reinterpret_cast<int32_t*>(keep + at.perm);
  int32_t* slot_pos = reinterpret_cast<int32_t*>(keep + at.slot_pos);
  void* rws = static_cast<char*>(workspace) + align256((size_t)N * E * 4);
  const size_t rws_bytes = align256(ygg_route_workspace_bytes(N, E, k));
  RowConvert cv;  // x's Pauli half-rows, in the routing's launches
  cv.x = x;
  cv.out = keep + at.x;
  cv.n = (long long)N * d;
  cv.d = d;
  cv.kind = kConvBf16Pauli;
  if (logits) {
    if (route_convert(logits, N, E, k, topk_idx, topk_w, counts, offsets, perm, slot_pos, rws, rws_bytes, cv, stream))
      return -1;
  } else if (route_energy_convert(x, kBF16, N, d, router_w, router_b, E, k, topk_idx, topk_w, counts, offsets, perm,
                                  slot_pos, static_cast<float*>(workspace), rws, rws_bytes, cv, stream)) {
    return -1;
  }
  if (pauli_linear_save_pre(keep + at.x, N, perm, P, w_up, b_up, offsets, E, d, F, act, keep + at.h, keep + at.h_pre, stream) ||
      ygg_pauli_grouped_linear(keep + at.h, /*Pauli rows*/ 1, P, nullptr, P, w_down, b_down, offsets, E, F, d, kActNone,
                               keep + at.y, /*blade*/ 1, kBF16, stream))
    return -1;
  return ygg_combine(keep + at.y, kBF16, /*y_mask=*/0, N, k, d, topk_idx, topk_w, slot_pos, residual, out, kBF16, stream);
}

YGG_API size_t ygg_moe_backward_bf16_workspace_bytes(int N, int d, int F, int E, int k) {
  if (N < 0 || d < 1 || F < 1 || E < 1 || k < 1 || (long long)N * k > 0x7fffffffLL) return 0;
  const size_t P = (size_t)N * k;
  return 2 * align256(P * d * 16) + align256(P * F * 16) +
         std::max(weight_grad_bf16_workspace_bytes((int)P, E, d, F), weight_grad_bf16_workspace_bytes((int)P, E, F, d));
}

YGG_API int ygg_moe_backward_bf16(int N, int d, int F, int E, int k, int act, const void* w_up_adj, const void* w_down_adj,
                                  int residual, const void* dout, const void* saved, size_t saved_bytes,
                                  const float* topk_w, const int32_t* offsets, void* dx, float* dw_up, float* db_up,
                                  float* dw_down, float* db_down, float* dtopk_w, void* workspace, size_t workspace_bytes,
                                  hipStream_t stream) {
  if (check_sizes("ygg_moe_backward_bf16", N, d, F, E, k, act)) return -1;
  YGG_CHECK_ARG(!dw_up == !db_up && !dw_down == !db_down,
                "ygg_moe_backward_bf16: null pointer (a weight's gradient and its bias's are given together or not at all)");
  if (N == 0) {  // no tokens: the weight and bias gradients are zero
    const size_t nw = (size_t)E * F * d * 8;
    return (dw_up && (fill_zero_f32(dw_up, nw, stream) || fill_zero_f32(db_up, (size_t)E * F * 8, stream))) ||
                   (dw_down && (fill_zero_f32(dw_down, nw, stream) || fill_zero_f32(db_down, (size_t)E * d * 8, stream)))
               ? -1 : 0;
  }
  YGG_CHECK_ARG(w_up_adj && w_down_adj && dout && saved && topk_w && offsets && dx && workspace,
                "ygg_moe_backward_bf16: null pointer");
  const Saved at = saved_of(N, d, F, k);
  YGG_CHECK_ARG(saved_bytes >= at.total, "ygg_moe_backward_bf16: %zu bytes of kept rows, need %zu", saved_bytes, at.total);
  const size_t need = ygg_moe_backward_bf16_workspace_bytes(N, d, F, E, k);
  YGG_CHECK_ARG(workspace_bytes >= need, "ygg_moe_backward_bf16: workspace of %zu bytes, need %zu", workspace_bytes, need);
  const int P = N * k;
  const char* const keep = static_cast<const char*>(saved);
  const int32_t* perm = reinterpret_cast<const int32_t*>(keep + at.perm);
  const int32_t* slot_pos = reinterpret_cast<const int32_t*>(keep + at.slot_pos);
  char* const dy = static_cast<char*>(workspace);
  char* const dxs = dy + align256((size_t)P * d * 16);
  char* const dh = dxs + align256((size_t)P * d * 16);
  void* const wg = dh + align256((size_t)P * F * 16);
  hipLaunchKernelGGL(combine_backward_bf16_kernel, dim3((N + 3) / 4), dim3(256), 0, stream,
                     static_cast<const uint16_t*>(dout),
                     dtopk_w ? reinterpret_cast<const uint16_t*>(keep + at.y) : nullptr, N, k, d, topk_w, slot_pos,
                     reinterpret_cast<uint16_t*>(dy), dtopk_w);
  if (check_launch("combine backward (bf16)")) return -1;
  if (ygg_pauli_grouped_input_grad(dy, P, w_down_adj, offsets, E, d, F, act, keep + at.h_pre, dh, /*Pauli rows*/ 0, kBF16,
                                   stream) ||
      (dw_down && weight_grad_bf16(dy, keep + at.h, P, nullptr, offsets, P, E, F, d, dw_down, db_down, wg, stream)) ||
      ygg_pauli_grouped_input_grad(dh, P, w_up_adj, offsets, E, F, d, kActNone, nullptr, dxs, /*blade*/ 1, kBF16, stream) ||
      (dw_up && weight_grad_bf16(dh, keep + at.x, N, perm, offsets, P, E, d, F, dw_up, db_up, wg, stream)))
    return -1;
  hipLaunchKernelGGL(dispatch_backward_bf16_kernel, dim3((unsigned)N), dim3(d <= 64 ? 64 : d <= 128 ? 128 : 256), 0, stream,
                     reinterpret_cast<const uint16_t*>(dxs), N, k, d, slot_pos,
                     residual ? static_cast<const uint16_t*>(dout) : nullptr, static_cast<uint16_t*>(dx));
  return check_launch("dispatch backward (bf16)");
}
