// weight_grad_bf16.hip -- the experts' weight and bias gradients from bf16 rows.
//
// For y_j = sum_i W_ji x_i + b_j (holograph/layers/clifford_linear.py:125-163, here per expert):
//   dW_ji = sum over the expert's rows r of dy_rj ~x_ri,   db_j = sum_r dy_rj
// In the Pauli coordinates of pauli_common.h reversion is the conjugate transpose, so dW_ji is
// the complex matrix sum_r M(dy_rj) M(x_ri)^H: C[a][c] = sum_{r, b} D_rj[a][b] conj(A_ri[c][b]).
// The rows are bf16 Pauli half-rows (rows, 2, d, 4), as the bf16 products read and write them:
// half b holds column b of every matrix, (re, im) of its entries 0 and 1.
//
// The sums are fp32 and their order depends on the sizes alone.

#include <hip/hip_runtime.h>

#include "pauli_common.h"
#include "ygg_common.h"

namespace ygg {
namespace {

constexpr int kRows = 8;   // rows staged at a time
constexpr int kTile = 32;  // columns j and i of a workgroup

// An expert's rows, whatever `offsets` holds: inside [0, P] and not negative
__device__ inline void expert_rows(const int32_t* __restrict__ offsets, int e, int P, int& r0, int& r1) {
  r0 = min(max(offsets[e], 0), P);
  r1 = max(min(offsets[e + 1], P), r0);
}

// Workgroup: a 32 (j) x 32 (i) tile of one expert; thread (tj, ti) the pairs (tj + 16 p, ti + 16 q).
__global__ __launch_bounds__(256) void weight_grad_bf16_kernel(const uint16_t* __restrict__ D,
                                                               const uint16_t* __restrict__ A, int a_rows,
                                                               const int32_t* __restrict__ gather,
                                                               const int32_t* __restrict__ offsets, int P, int d_in,
                                                               int d_out, float* __restrict__ dW,
                                                               float* __restrict__ db) {
  __shared__ float4 sd[kRows][kTile][2], sa[kRows][kTile][2];  // columns b = 0, 1: re, im of entries 0 and 1
  const int e = blockIdx.z, j0 = blockIdx.x * kTile, i0 = blockIdx.y * kTile;
  const int tid = threadIdx.x, tj = tid & 15, ti = tid >> 4;
  int r0, r1;
  expert_rows(offsets, e, P, r0, r1);
  float acc[2][2][8] = {}, bsum[8] = {};  // [p][q][a c re/im]; this thread's staged rows of dy
  const int sr = tid >> 5, sc = tid & 31;
  auto stage = [&](const uint16_t* rows, long long row, int d, int col, float4 (&to)[kRows][kTile][2]) {
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
      if (row >= 0 && col < d) {
        const uint2 q = *reinterpret_cast<const uint2*>(rows + (((size_t)row * 2 + b) * d + col) * 4);
        v = make_float4(bf_lo(q.x), bf_hi(q.x), bf_lo(q.y), bf_hi(q.y));
      }
      to[sr][sc][b] = v;
    }
  };
  for (int base = r0; base < r1; base += kRows) {
    const int r = base + sr;
    const int src = r < r1 ? (gather ? gather[r] : r) : -1;
    stage(D, r < r1 ? r : -1, d_out, j0 + sc, sd);
    stage(A, src >= 0 && src < a_rows ? src : -1, d_in, i0 + sc, sa);
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      const float4 v = sd[sr][sc][b];
      bsum[4 * b] += v.x; bsum[4 * b + 1] += v.y; bsum[4 * b + 2] += v.z; bsum[4 * b + 3] += v.w;
    }
    __syncthreads();
    for (int rr = 0; rr < min(kRows, r1 - base); ++rr)
#pragma unroll
      for (int p = 0; p < 2; ++p)
#pragma unroll
        for (int q = 0; q < 2; ++q)
#pragma unroll
          for (int b = 0; b < 2; ++b) {
            const float4 u = sd[rr][tj + 16 * p][b], v = sa[rr][ti + 16 * q][b];
            float* s = acc[p][q];
            s[0] += u.x * v.x + u.y * v.y;  s[1] += u.y * v.x - u.x * v.y;  // a = 0, c = 0
            s[2] += u.x * v.z + u.y * v.w;  s[3] += u.y * v.z - u.x * v.w;  // a = 0, c = 1
            s[4] += u.z * v.x + u.w * v.y;  s[5] += u.w * v.x - u.z * v.y;  // a = 1, c = 0
            s[6] += u.z * v.z + u.w * v.w;  s[7] += u.w * v.z - u.z * v.w;  // a = 1, c = 1
          }
    __syncthreads();
  }
  auto store = [](float* dst, const float* s) {  // half the blades of the summed matrix
    float o[8];
    pauli_to_blade(s[0], s[1], s[2], s[3], s[4], s[5], s[6], s[7], o);
    float4* q = reinterpret_cast<float4*>(dst);
    q[0] = make_float4(0.5f * o[0], 0.5f * o[1], 0.5f * o[2], 0.5f * o[3]);
    q[1] = make_float4(0.5f * o[4], 0.5f * o[5], 0.5f * o[6], 0.5f * o[7]);
  };
#pragma unroll
  for (int p = 0; p < 2; ++p)
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const int j = j0 + tj + 16 * p, i = i0 + ti + 16 * q;
      if (j < d_out && i < d_in) store(dW + (((size_t)e * d_out + j) * d_in + i) * 8, acc[p][q]);
    }
  if (db != nullptr && blockIdx.y == 0) {
    float* red = reinterpret_cast<float*>(&sd[0][0][0]);
#pragma unroll
    for (int c = 0; c < 8; ++c) red[(sr * kTile + sc) * 8 + c] = bsum[c];
    __syncthreads();
    if (sr == 0 && j0 + sc < d_out) {
      float s[8] = {};
      for (int q = 0; q < kRows; ++q)
#pragma unroll
        for (int c = 0; c < 8; ++c) s[c] += red[(q * kTile + sc) * 8 + c];
      // columns (entry 0, entry 1) b = 0, 1 -> M00, M01, M10, M11
      const float m[8] = {s[0], s[1], s[4], s[5], s[2], s[3], s[6], s[7]};
      store(db + ((size_t)e * d_out + j0 + sc) * 8, m);
    }
  }
}

}  // namespace

size_t weight_grad_bf16_workspace_bytes(int P_max, int E, int d_in, int d_out) { return 0; }

int weight_grad_bf16(const void* dy, const void* a, int a_rows, const int32_t* gather, const int32_t* offsets, int P_max,
                     int E, int d_in, int d_out, float* dW, float* db, void* workspace, hipStream_t stream) {
  if (E == 0) return 0;
  hipLaunchKernelGGL(weight_grad_bf16_kernel, dim3((d_out + kTile - 1) / kTile, (d_in + kTile - 1) / kTile, E), dim3(256),
                     0, stream, static_cast<const uint16_t*>(dy), static_cast<const uint16_t*>(a), a_rows, gather,
                     offsets, P_max, d_in, d_out, dW, db);
  return check_launch("weight gradient (bf16)");
}

}  // namespace ygg

using namespace ygg;

YGG_API size_t ygg_grouped_weight_grad_pauli_bf16_workspace_bytes(int P_max, int E, int d_in, int d_out) {
  if (P_max < 0 || E < 0 || d_in < 1 || d_out < 1) return 0;
  return weight_grad_bf16_workspace_bytes(P_max, E, d_in, d_out);
}

YGG_API int ygg_grouped_weight_grad_pauli_bf16(const void* dy_pauli, const void* a_pauli, int a_rows,
                                               const int32_t* gather, const int32_t* offsets, int P_max, int E, int d_in,
                                               int d_out, float* dW, float* db, void* workspace, size_t workspace_bytes,
                                               hipStream_t stream) {
  YGG_CHECK_ARG(P_max >= 0 && E >= 0 && E <= 64 && d_in >= 2 && d_in % 2 == 0 && d_out >= 2 && d_out % 2 == 0,
                "ygg_grouped_weight_grad_pauli_bf16: bad sizes P_max=%d E=%d d_in=%d d_out=%d (E <= 64, even d_in and "
                "d_out)", P_max, E, d_in, d_out);
  YGG_CHECK_ARG(a_rows >= 0 && (gather != nullptr || a_rows >= P_max),
                "ygg_grouped_weight_grad_pauli_bf16: a has %d rows, %d are read without a gather", a_rows, P_max);
  if (E == 0) return 0;
  YGG_CHECK_ARG(offsets && dW && (P_max == 0 || (dy_pauli && a_pauli)),
                "ygg_grouped_weight_grad_pauli_bf16: null pointer argument");
  const size_t need = weight_grad_bf16_workspace_bytes(P_max, E, d_in, d_out);
  YGG_CHECK_ARG(need == 0 || (workspace && workspace_bytes >= need),
                "ygg_grouped_weight_grad_pauli_bf16: workspace of %zu bytes, need %zu", workspace ? workspace_bytes : 0,
                need);
  return weight_grad_bf16(dy_pauli, a_pauli, a_rows, gather, offsets, P_max, E, d_in, d_out, dW, db, workspace, stream);
}
