// sort_backward.hip -- the gradients of the sort by expert and of the weighted way back (hlm_block.py:178, 180-181;
// forward: dispatch.hip; the reference has no MoE backward, hlm_block.py:202-206).
//
//   out_t = sum_s w_ts y[slot_ts]:   dy[slot_ts] = w_ts dout_t,   dw_ts = <dout_t, y[slot_ts]>
//   x_sorted[slot_ts] = x_t:         dx_t = sum_s dx_sorted[slot_ts]  (and what reaches x_t past the sort)
//
// Every row is read once and written once: both are bound by memory.  A slot names one row, so nothing is added
// across workgroups; a token's rows are added in slot order, in fp32.  A slot outside the rows is left out, and a row
// that no slot names has the gradient zero.

#include <hip/hip_runtime.h>

#include <algorithm>

#include "rows.h"
#include "ygg_common.h"

namespace ygg {
namespace {

constexpr int kMaxTopK = 8;
constexpr int kLaunchTokens = 1 << 22;  // tokens of a launch: a grid holds fewer than 2^32 threads

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

// Rows that no slot names get the gradient zero.  They are found in one of two ways, neither of which needs memory to be
// cleared first:
//   few slots and rows: workgroups in front of the tokens' own, kFindRows rows each, look through every slot;
//   else a launch behind the tokens', which left in row_token the token of each named row (and of the others whatever the
//   memory held): a row is named if the token that stands there has a slot that names it.
// The first costs no launch and no scratch, but P N k / kFindRows reads (what finding adds, first / second way, us: 512 slots
// and rows 0.8 / 3.5, 8192: 0.1, 16384: 1.5 / 2.4, 32768: 3.1 / 2.6, 131072: 12 to 30 / 3.9).
constexpr int kFindRows = 512;
constexpr long long kFindMost = 1LL << 28;  // P N k
bool finds_by_slots(int N, int k, int P) { return N <= kLaunchTokens && (long long)N * k <= kFindMost / std::max(P, 1); }

// the rows of a wave's lanes that are not named, from row `first` on, cleared by the wave
__device__ __forceinline__ void clear_rows(bool named, size_t first, int row_pieces, uint4* __restrict__ dy) {
  for (uint64_t left = __ballot(!named); left != 0; left &= left - 1) {
    uint4* const to = dy + (first + __builtin_ctzll(left)) * row_pieces;
    for (int i = threadIdx.x & 63; i < row_pieces; i += 64) to[i] = make_uint4(0, 0, 0, 0);
  }
}
__device__ __forceinline__ void find_and_clear(const int32_t* __restrict__ slot_pos, size_t slots, int P, int row_pieces,
                                               uint4* __restrict__ dy) {
  __shared__ unsigned char s_named[kFindRows];
  const int row0 = blockIdx.x * kFindRows;
  for (int r = threadIdx.x; r < kFindRows; r += 256) s_named[r] = r >= P - row0;
  __syncthreads();
  typedef int i4_t __attribute__((ext_vector_type(4), aligned(4)));
  auto mark = [&](int at) {
    if (at >= row0 && at < P && at - row0 < kFindRows) s_named[at - row0] = 1;
  };
  const size_t fours = slots / 4;
#pragma unroll 4
  for (size_t q = threadIdx.x; q < fours; q += 256) {
    const i4_t at = reinterpret_cast<const i4_t*>(slot_pos)[q];
#pragma unroll
    for (int c = 0; c < 4; ++c) mark(at[c]);
  }
  if (fours * 4 + threadIdx.x < slots) mark(slot_pos[fours * 4 + threadIdx.x]);
  __syncthreads();
  const int wave = threadIdx.x >> 6;
  for (int r = wave * 64; r < kFindRows; r += 256) clear_rows(s_named[r + (threadIdx.x & 63)], (size_t)row0 + r, row_pieces, dy);
}

// One wave per token (bf16 half-rows, 8192 tokens, d = 128, k = 4: 25.7 us, 151 MB that the last-level cache holds in part;
// 131072 tokens: 474 us with the search above, 2.4 GB at 5.1 TB/s).
template <typename TD, typename TY, int LAYOUT>
__global__ __launch_bounds__(256) void combine_backward_kernel(const TD* __restrict__ dout, const TY* __restrict__ y, int N,
                                                               int k, int d, int P, const float* __restrict__ topk_w,
                                                               const int32_t* __restrict__ slot_pos, TY* __restrict__ dy,
                                                               float* __restrict__ dtopk_w, unsigned finders,
                                                               int32_t* __restrict__ row_token, int first) {
  if (blockIdx.x < finders) {
    find_and_clear(slot_pos, (size_t)N * k, P, d * (int)sizeof(TY) / 2, reinterpret_cast<uint4*>(dy));
    return;
  }
  const int lane = threadIdx.x & 63;
  const int t = (blockIdx.x - finders) * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (t >= N) return;
  if (row_token != nullptr && lane < k) {
    const int at = slot_pos[(size_t)t * k + lane];
    if ((unsigned)at < (unsigned)P) row_token[at] = first + t;
  }
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

__global__ __launch_bounds__(256) void clear_unnamed_kernel(const int32_t* __restrict__ row_token,
                                                            const int32_t* __restrict__ slot_pos, int N, int k, int P,
                                                            int row_pieces, uint4* __restrict__ dy) {
  const size_t first = ((size_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6)) * 64;
  const size_t row = first + (threadIdx.x & 63);
  bool named = row >= (size_t)P;
  if (!named) {
    const int t = row_token[row];
    if ((unsigned)t < (unsigned)N)
      for (int s = 0; s < k; ++s) named = named || slot_pos[(size_t)t * k + s] == (int)row;
  }
  clear_rows(named, first, row_pieces, dy);
}

// A thread per multivector of a token (bf16, 8192 tokens, d = 128, k = 4: 17.6 us, 84 MB; 131072 tokens: 250 us, 1.3 GB at 5.4
// TB/s).
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

template <typename TD, typename TY>
int launch_combine(const void* dout, const void* y, int N, int k, int d, int P, const float* w, const int32_t* slots, void* dy,
                   int layout, float* dw, bool whole, int32_t* row_token, hipStream_t stream) {
  const unsigned finders = whole && !row_token ? (unsigned)(((size_t)P + kFindRows - 1) / kFindRows) : 0;
  const TY* Y = static_cast<const TY*>(y);
  TY* O = static_cast<TY*>(dy);
  // (no tokens: the finders alone; finders look through one launch's slots, finds_by_slots)
  for (size_t t0 = 0; t0 < (size_t)N || (t0 == 0 && finders); t0 += kLaunchTokens) {
    const int n = (int)std::min<size_t>(N - t0, kLaunchTokens);
    const unsigned grid = (unsigned)(n + 3) / 4;
    const TD* const D = static_cast<const TD*>(dout) + t0 * d * 8;
    const float* const W = w + t0 * k;
    const int32_t* const S = slots + t0 * k;
    float* const DW = dw ? dw + t0 * k : nullptr;
    auto* const kernel = layout == kDyPauli ? combine_backward_kernel<TD, TY, kDyPauli> : combine_backward_kernel<TD, TY, kDyBlade>;
    kernel<<<grid + finders, 256, 0, stream>>>(D, Y, n, k, d, P, W, S, O, DW, finders, row_token, (int)t0);
    if (check_launch("combine_backward")) return -1;
  }
  if (row_token == nullptr) return 0;
  clear_unnamed_kernel<<<(unsigned)(((size_t)P + 255) / 256), 256, 0, stream>>>(row_token, slots, N, k, P,
                                                                                d * (int)sizeof(TY) / 2, reinterpret_cast<uint4*>(O));
  return check_launch("combine_backward (rows that no slot names)");
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
  return launch_combine<uint16_t, uint16_t>(dout, y, N, k, d, N * k, topk_w, slot_pos, dy, kDyPauli, dtopk_w, false, nullptr, stream);
}

int dispatch_backward_bf16(const void* dxs, int N, int k, int d, const int32_t* slot_pos, const void* add, void* dx,
                           hipStream_t stream) {
  return launch_dispatch<uint16_t>(dxs, N, k, d, N * k, slot_pos, add, dx, stream);
}

}  // namespace ygg

using namespace ygg;

static int run_combine_backward(const char* who, const void* dout, int dout_dtype, const void* y_sorted, int N, int k, int d,
                                int P, const float* topk_w, const int32_t* slot_pos, void* dy, int dy_dtype, int dy_layout,
                                float* dtopk_w, bool whole, int32_t* row_token, hipStream_t stream) {
  YGG_CHECK_ARG(N >= 0 && d >= 1 && k >= 1 && k <= kMaxTopK && P >= 0, "%s: bad sizes N=%d k=%d d=%d P=%d (k <= %d)",
                who, N, k, d, P, kMaxTopK);
  YGG_CHECK_ARG((dout_dtype == kF32 || dout_dtype == kBF16) && (dy_dtype == kF32 || dy_dtype == kBF16),
                "%s: dtypes %d, %d unsupported", who, dout_dtype, dy_dtype);
  YGG_CHECK_ARG(dy_layout == kDyBlade || dy_layout == kDyPauli, "%s: layout %d", who, dy_layout);
  if (N == 0 && (!whole || P == 0)) return 0;
  YGG_CHECK_ARG((N == 0 || (dout && topk_w && slot_pos)) && (dy || P == 0), "%s: null pointer", who);
  YGG_CHECK_ARG(N == 0 || !y_sorted == !dtopk_w || (P == 0 && dtopk_w),
                "%s: the routing weights' gradient needs y_sorted, and y_sorted it", who);
  const size_t db = (size_t)N * d * 8 * dtype_size(dout_dtype), yb = (size_t)P * d * 8 * dtype_size(dy_dtype);
  const size_t slots = (size_t)N * k * 4, tokens = (size_t)P * 4;
  YGG_CHECK_ARG(!overlap(dy, yb, dout, db) && !overlap(dy, yb, y_sorted, yb) && !overlap(dy, yb, topk_w, slots) &&
                    !overlap(dy, yb, slot_pos, slots) && !overlap(dy, yb, dtopk_w, slots) && !overlap(dtopk_w, slots, dout, db) &&
                    !overlap(dtopk_w, slots, y_sorted, yb) && !overlap(dtopk_w, slots, topk_w, slots) &&
                    !overlap(dtopk_w, slots, slot_pos, slots) && !overlap(row_token, tokens, dout, db) &&
                    !overlap(row_token, tokens, y_sorted, yb) && !overlap(row_token, tokens, topk_w, slots) &&
                    !overlap(row_token, tokens, slot_pos, slots) && !overlap(row_token, tokens, dy, yb) &&
                    !overlap(row_token, tokens, dtopk_w, slots),
                "%s: outputs must not share memory with inputs or each other", who);
  if (dout_dtype == kF32)
    return dy_dtype == kF32
               ? launch_combine<float, float>(dout, y_sorted, N, k, d, P, topk_w, slot_pos, dy, dy_layout, dtopk_w, whole, row_token, stream)
               : launch_combine<float, uint16_t>(dout, y_sorted, N, k, d, P, topk_w, slot_pos, dy, dy_layout, dtopk_w, whole, row_token, stream);
  return dy_dtype == kF32
             ? launch_combine<uint16_t, float>(dout, y_sorted, N, k, d, P, topk_w, slot_pos, dy, dy_layout, dtopk_w, whole, row_token, stream)
             : launch_combine<uint16_t, uint16_t>(dout, y_sorted, N, k, d, P, topk_w, slot_pos, dy, dy_layout, dtopk_w, whole, row_token, stream);
}

YGG_API int ygg_combine_backward(const void* dout, int dout_dtype, const void* y_sorted, int N, int k, int d, int P,
                                 const float* topk_w, const int32_t* slot_pos, void* dy, int dy_dtype, int dy_layout,
                                 float* dtopk_w, hipStream_t stream) {
  return run_combine_backward("ygg_combine_backward", dout, dout_dtype, y_sorted, N, k, d, P, topk_w, slot_pos, dy, dy_dtype,
                              dy_layout, dtopk_w, false, nullptr, stream);
}

YGG_API size_t ygg_combine_backward_rows_workspace_bytes(int N, int k, int P) {
  return N < 0 || k < 1 || P < 0 || finds_by_slots(N, k, P) ? 0 : (size_t)P * 4;
}

YGG_API int ygg_combine_backward_rows(const void* dout, int dout_dtype, const void* y_sorted, int N, int k, int d, int P,
                                      const float* topk_w, const int32_t* slot_pos, void* dy, int dy_dtype, int dy_layout,
                                      float* dtopk_w, void* workspace, size_t workspace_bytes, hipStream_t stream) {
  const size_t need = ygg_combine_backward_rows_workspace_bytes(N, k, P);
  YGG_CHECK_ARG(need == 0 || (workspace && workspace_bytes >= need),
                "ygg_combine_backward_rows: workspace of %zu bytes, need %zu", workspace ? workspace_bytes : (size_t)0, need);
  return run_combine_backward("ygg_combine_backward_rows", dout, dout_dtype, y_sorted, N, k, d, P, topk_w, slot_pos, dy,
                              dy_dtype, dy_layout, dtopk_w, true, need ? static_cast<int32_t*>(workspace) : nullptr, stream);
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
