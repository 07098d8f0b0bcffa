// rows.h -- multivectors of fp32 and bf16 blade-order rows, and sums over a wave, shared by the
// gradients that are bound by memory (norm_backward.hip, route_backward.hip).
#pragma once

#include "pauli_common.h"

namespace ygg {

// one multivector as it is stored: the loads of a batch are issued before the first is unpacked
template <typename T>
struct RawMv;
template <>
struct RawMv<float> {
  float4 a, b;
};
template <>
struct RawMv<uint16_t> {
  uint4 a;
};
__device__ __forceinline__ RawMv<float> load_raw(const float* p, size_t n) {
  const float4* q = reinterpret_cast<const float4*>(p + n * 8);
  return RawMv<float>{q[0], q[1]};
}
__device__ __forceinline__ RawMv<uint16_t> load_raw(const uint16_t* p, size_t n) {
  return RawMv<uint16_t>{*reinterpret_cast<const uint4*>(p + n * 8)};
}
__device__ __forceinline__ void unpack(const RawMv<float>& m, float v[8]) {
  v[0] = m.a.x; v[1] = m.a.y; v[2] = m.a.z; v[3] = m.a.w;
  v[4] = m.b.x; v[5] = m.b.y; v[6] = m.b.z; v[7] = m.b.w;
}
__device__ __forceinline__ void unpack(const RawMv<uint16_t>& m, float v[8]) {
  v[0] = bf_lo(m.a.x); v[1] = bf_hi(m.a.x); v[2] = bf_lo(m.a.y); v[3] = bf_hi(m.a.y);
  v[4] = bf_lo(m.a.z); v[5] = bf_hi(m.a.z); v[6] = bf_lo(m.a.w); v[7] = bf_hi(m.a.w);
}
template <typename T>
__device__ __forceinline__ void load_mv(const T* p, size_t n, float v[8]) {
  unpack(load_raw(p, n), v);
}
__device__ __forceinline__ void store_mv(float* p, size_t n, const float v[8]) {
  float4* q = reinterpret_cast<float4*>(p + n * 8);
  q[0] = make_float4(v[0], v[1], v[2], v[3]);
  q[1] = make_float4(v[4], v[5], v[6], v[7]);
}
__device__ __forceinline__ void store_mv(uint16_t* p, size_t n, const float v[8]) {
  *reinterpret_cast<uint4*>(p + n * 8) =
      make_uint4(pack2_bf16(v[0], v[1]), pack2_bf16(v[2], v[3]), pack2_bf16(v[4], v[5]), pack2_bf16(v[6], v[7]));
}

// V values (a power of two) summed over the wave with V + log2(64 / V) - 1 exchanges in the place of 6 V: each
// of the first steps halves the values that a lane carries on.  Returns the sum of value wave_sums_of(lane).
// (By recursion: as loops over n and o, 16 values were indexed at run time.)
template <int V, int N = V / 2, int O = 32>
__device__ __forceinline__ float wave_sums(float (&v)[V], int lane) {
  if constexpr (N > 0) {
    const bool up = (lane & O) != 0;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float keep = up ? v[i + N] : v[i], give = up ? v[i] : v[i + N];
      v[i] = keep + __shfl_xor(give, O);
    }
    return wave_sums<V, N / 2, O / 2>(v, lane);
  } else if constexpr (O > 0) {
    v[0] += __shfl_xor(v[0], O);
    return wave_sums<V, 0, O / 2>(v, lane);
  }
  return v[0];
}
// the value whose sum the lane holds: bit 5 of the lane chose between the halves, bit 4 between their halves, ...
template <int V>
__device__ __forceinline__ int wave_sums_of(int lane) {
  return V == 1 ? 0 : lane / (64 / V);
}

// Planes of `values` floats added, by a workgroup of 1024: 32 values, 32 threads for each -- a thread every
// 32nd plane in order, their sums as a tree -- and out(n, sum of value n).
template <class F>
__device__ __forceinline__ void add_planes(const float* __restrict__ part, int planes, int values, F&& out) {
  __shared__ float red[32][33];
  const int v = threadIdx.x & 31, k = threadIdx.x >> 5, n = blockIdx.x * 32 + v;
  float s = 0.f;
  if (n < values) {
#pragma unroll 8
    for (int p = k; p < planes; p += 32) s += part[(size_t)p * values + n];
  }
  red[k][v] = s;
  __syncthreads();
  float t = red[v][k];  // of value k, the sum of thread v
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) t += __shfl_xor(t, o);
  const int m = blockIdx.x * 32 + k;
  if (v == 0 && m < values) out(m, t);
}

}  // namespace ygg
