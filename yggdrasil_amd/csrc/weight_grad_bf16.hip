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

#include <algorithm>
#include <type_traits>

#include "pauli_split.h"
#include "ygg_common.h"

namespace ygg {
namespace {

constexpr int kWbTile = 64;     // output columns j and input columns i of a workgroup
constexpr int kWbRows = 12;      // rows of a stage
constexpr int kWbStages = 3;    // stages in LDS: two in flight while one is read
constexpr int kWbWaveRows = kWbRows / 4;  // rows that a wave loads per stage
constexpr int kWbMaxChunk = 1024, kWbMinChunk = 256;  // rows of a workgroup at most, see chunk_rows
constexpr int kWbHalf = kWbTile * 8;               // bytes of a half-row of a stage
constexpr int kWbOperand = kWbRows * 2 * kWbHalf;  // bytes of one operand of a stage
constexpr int kWbStage = 2 * kWbOperand;

// Inclusive scans over the wave by DPP moves (rows of 16 lanes, then each row's last lane to the next rows): a
// quarter of the latency of six exchanges through LDS, of which a workgroup waits for three one after another.
template <bool MAX>
__device__ __forceinline__ int wave_scan(int v) {
  auto step = [&](auto ctrl, auto rows) __attribute__((always_inline)) {
    const int u = __builtin_amdgcn_update_dpp(MAX ? v : 0, v, decltype(ctrl)::value, decltype(rows)::value, 0xf, false);
    v = MAX ? max(v, u) : v + u;
  };
  typedef std::integral_constant<int, 0xf> all;
  step(std::integral_constant<int, 0x111>{}, all{});  // row_shr:1, 2, 4, 8
  step(std::integral_constant<int, 0x112>{}, all{});
  step(std::integral_constant<int, 0x114>{}, all{});
  step(std::integral_constant<int, 0x118>{}, all{});
  step(std::integral_constant<int, 0x142>{}, std::integral_constant<int, 0xa>{});  // row_bcast:15 into rows 1 and 3
  step(std::integral_constant<int, 0x143>{}, std::integral_constant<int, 0xc>{});  // row_bcast:31 into rows 2 and 3
  return v;
}

// Lane e: the rows of expert e and their chunks, n = ceil(rows / limit) of equal length (a multiple of a
// stage's rows).  Whatever `offsets` holds, the ranges are inside [0, P] and disjoint: every bound is
// clamped and at least the one before it.
struct WbExpert {
  int beg, end, n, len;
};
__device__ __forceinline__ WbExpert wb_experts(const int32_t* __restrict__ offsets, int E, int P, int limit,
                                               int lane) {
  const int beg = wave_scan<true>(min(max(offsets[min(lane, E)], 0), P));
  WbExpert x = {beg, max(beg, min(offsets[min(lane + 1, E)], P)), 0, 0};
  if (lane >= E) x.end = x.beg;
  x.n = (x.end - x.beg + limit - 1) / limit;
  x.len = x.n > 0 ? ((x.end - x.beg + x.n - 1) / x.n + kWbRows - 1) / kWbRows * kWbRows : 0;
  return x;
}

__device__ __forceinline__ float swap_pair(float v) {  // the value of the neighbouring lane (lane ^ 1)
  return __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), 0xB1, 0xf, 0xf, true));
}
// From this lane's half of a summed matrix -- lane parity c: entries (0, c) and (1, c), re and im -- and its
// neighbour's, four values of half its blades: blades 0 to 3 for c = 0, 4 to 7 for c = 1.
__device__ __forceinline__ float4 half_blades(float r0, float i0, float r1, float i1, int c) {
  const float x = swap_pair(c ? r1 : i0), y = swap_pair(c ? r0 : r1), z = swap_pair(c ? i0 : i1);
  return c ? make_float4(0.5f * (x - i1), 0.5f * (y - r0), 0.5f * (z + i0), 0.5f * (x + i1))
           : make_float4(0.5f * (r0 + x), 0.5f * (r1 + y), 0.5f * (i1 - z), 0.5f * (r0 - x));
}

// A tile of the gradient of expert e, which has no rows
__device__ __forceinline__ void zero_tile(int jt, int it, int e, int d_in, int d_out, float* __restrict__ dW,
                                          float* __restrict__ db, int tid) {
  const float4 z = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int n = tid; n < kWbTile * kWbTile * 2; n += 256) {
    const int j = jt * kWbTile + n / (kWbTile * 2), i2 = it * kWbTile * 2 + n % (kWbTile * 2);
    if (j < d_out && i2 < d_in * 2) reinterpret_cast<float4*>(dW)[((size_t)e * d_out + j) * d_in * 2 + i2] = z;
  }
  if (db != nullptr && it == 0 && tid < kWbTile * 2 && jt * kWbTile * 2 + tid < d_out * 2)
    reinterpret_cast<float4*>(db)[(size_t)e * d_out * 2 + jt * kWbTile * 2 + tid] = z;
}

// One workgroup: 64 (j) x 64 (i) of one chunk's sum, a wave 32 x 32 of it.
//
// Bound by the matrix units and the loads into LDS together: 8192 tokens, d = 128, F = 512, E = 32, k = 4, Zipf's
// law take 153-157 us in all, 131-142 here and 15-16 in the planes' sum: 137 GFLOP at 1.0 PFLOP/s here, where a large
// bf16 product reaches 1.37.  The matrix units are busy 47 % of the time: of the two waves that a SIMD holds 1.4 are there
// on average, as the chunks of uneven experts do not end together.  (Variants, against 159 in all at their time:) without
// the loads (data in LDS as it was) 137 us, without the products 133.  Larger tiles did not pay: 128 x 64 with eight waves
// 160 us, with four waves of 64 x 32, one a SIMD, 179; nor did eight waves on one tile, half of a chunk's rows each (157,
// and half the planes, but one tile a CU: 1500 ragged tokens as below 26-30 us against 27), reading the next stage's
// operands into registers ahead (160) or raising the waves' priority (174).
//
// v_mfma_f32_32x32x16_bf16 with the operand rows (j, a) and columns (i, c), 16 of each index: the dword
// (re, im) of entry a of column b of D_rj is one (r, b) term of the contraction, and four such dwords (two
// rows, b = 0, 1) are a lane's operand.  D . A sums re re + im im, the real part of D conj(A); with A rotated
// to (im, -re) the sum is minus the imaginary part.  The dwords of 32 operand rows are neighbours in a
// half-row, so the LDS reads, four times 4 bytes per operand, are free of bank conflicts without padding.
//
// The rows come by direct-to-LDS loads, 16 bytes a lane, one row of 64 columns an instruction.  Rows in place
// are addressed from the chunk's first one (64-bit base: operands of any size); gathered rows over the whole
// of A, which the host keeps below 2 GiB.
template <bool GATHER>
__global__ __launch_bounds__(256, 2) void weight_grad_bf16_kernel(
    const uint16_t* __restrict__ D, const uint16_t* __restrict__ A, int a_rows, const int32_t* __restrict__ gather_rows,
    const int32_t* __restrict__ offsets, int P, int limit, int E, int d_in, int d_out, int n_xcd, float* __restrict__ part,
    float* __restrict__ dbpart, float* __restrict__ dW, float* __restrict__ db) {
  __shared__ __attribute__((aligned(1024))) unsigned char smem[kWbStages * kWbStage];
  __shared__ uint32_t s_src[GATHER ? kWbMaxChunk + kWbRows * (kWbStages + 1) : 1];
  const int32_t* const gather = GATHER ? gather_rows : nullptr;
  const int tid = threadIdx.x, lane = tid & 63;
  const int nj = (d_out + kWbTile - 1) / kWbTile, ni = (d_in + kWbTile - 1) / kWbTile, nt = nj * ni;
  // all tiles of a chunk on one XCD (workgroup b runs on XCD b mod 8): its rows are read into one L2.  The chunks
  // fall in length, so every second round of them goes over the XCDs backwards (Zipf's law as above: 162 -> 159 us).
  const int bq = blockIdx.x / n_xcd, round = bq / nt, tile = bq - round * nt, xcd = blockIdx.x - bq * n_xcd;
  const int chunk = round * n_xcd + ((round & 1) ? n_xcd - 1 - xcd : xcd);
  const WbExpert x = wb_experts(offsets, E, P, limit, lane);
  // the chunks in order of falling length, so that the last to start are short: this lane's expert's first one
  const int planes = wave_scan<false>(x.n > 1 ? x.n : 0), key = x.len * 64 + 63 - lane;
  int first = 0;
  for (int i = 0; i < E; ++i) {
    const int k = __builtin_amdgcn_readlane(key, i), m = __builtin_amdgcn_readlane(x.n, i);
    first += k > key ? m : 0;
  }
  const uint64_t mine = __ballot(lane < E && chunk >= first && chunk < first + x.n);
  if (mine == 0) {  // behind the chunks: the experts without rows, whose gradient is zero
    const uint64_t none = __ballot(lane < E && x.n == 0);
    const int total = __builtin_amdgcn_readlane(wave_scan<false>(x.n), 63);
    const int nth = __popcll(none & ((1ull << lane) - 1));  // this lane's place among them
    const uint64_t here = __ballot(lane < E && x.n == 0 && nth == chunk - total);
    if (here != 0) zero_tile(tile % nj, tile / nj, (int)__builtin_ctzll(here), d_in, d_out, dW, db, tid);
    return;
  }
  const int e = (int)__builtin_ctzll(mine);
  const int n = __builtin_amdgcn_readlane(x.n, e), c = chunk - __builtin_amdgcn_readlane(first, e);
  const int len = __builtin_amdgcn_readlane(x.len, e);
  const int r0 = __builtin_amdgcn_readlane(x.beg, e) + c * len;
  const int rows = max(0, min(len, __builtin_amdgcn_readlane(x.end, e) - r0));
  const int plane = __builtin_amdgcn_readlane(planes, e) - n + c;  // of an expert of several chunks
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int j0 = (tile % nj) * kWbTile, i0 = (tile / nj) * kWbTile;

  // the byte offset of every row's A from a_rsrc's base, or one past any range
  const uint32_t a_row = (uint32_t)d_in * 16;
  if (gather != nullptr)
    for (int i = tid; i < limit + kWbRows * (kWbStages + 1); i += 256) {
      const int src = i < rows ? gather[r0 + i] : -1;
      s_src[i] = src >= 0 && src < a_rows ? (uint32_t)src * a_row : kBufferOff;
    }
  __syncthreads();

  // A row past the chunk lies past its descriptor's range and reads zeros.  This lane's piece of a row:
  // half lane / 32, columns 2 (lane % 32) and the next; columns past the width get an offset past any range.
  const __amdgpu_buffer_rsrc_t d_rsrc = __builtin_amdgcn_make_buffer_rsrc(
      const_cast<uint16_t*>(D) + (size_t)r0 * d_out * 8, (short)0, (uint32_t)rows * d_out * 16, kBufferFlags);
  const __amdgpu_buffer_rsrc_t a_rsrc = __builtin_amdgcn_make_buffer_rsrc(
      const_cast<uint16_t*>(A) + (gather ? 0 : (size_t)r0 * d_in * 8), (short)0, (uint32_t)(gather ? a_rows : rows) * a_row,
      kBufferFlags);
  const int col = 2 * (lane & 31);
  const uint32_t d_bad = j0 + col < d_out ? 0u : kBufferOff, a_bad = i0 + col < d_in ? 0u : kBufferOff;
  const uint32_t a_lane = (uint32_t)((lane >> 5) * d_in + i0 + col) * 8;
  uint32_t d_next = (uint32_t)((lane >> 5) * d_out + j0 + col) * 8 + (uint32_t)(kWbWaveRows * wave) * d_out * 16;
  uint32_t a_next = a_lane + (uint32_t)(kWbWaveRows * wave) * a_row;  // (rows in place)
  const uint32_t lds0 = (uint32_t)(uintptr_t)(sp_lds_t*)smem + kWbWaveRows * wave * 2 * kWbHalf;
  uint32_t src[kWbWaveRows] = {};  // gathered: the offsets of the next stage's rows
  auto next_src = [&](int f) __attribute__((always_inline)) {
    if constexpr (GATHER) {
#pragma unroll
      for (int u = 0; u < kWbWaveRows; ++u) src[u] = s_src[f * kWbRows + kWbWaveRows * wave + u];
    }
  };
  auto issue = [&](int f) __attribute__((always_inline)) {  // stage f's rows, three of each operand a wave
    const uint32_t st = lds0 + (f % kWbStages) * kWbStage;
#pragma unroll
    for (int u = 0; u < kWbWaveRows; ++u) {
      split_dma(d_rsrc, st + u * 2 * kWbHalf, (d_next + u * (uint32_t)d_out * 16) | d_bad, 0);
      split_dma(a_rsrc, st + kWbOperand + u * 2 * kWbHalf, (GATHER ? src[u] + a_lane : a_next + u * a_row) | a_bad, 0);
    }
    d_next += (uint32_t)kWbRows * d_out * 16;
    a_next += (uint32_t)kWbRows * a_row;
  };
  const int wj = wave & 1, wi = wave >> 1, l32 = lane & 31, g = lane >> 5;
  // (bases that the compiler cannot relate, so that it pairs the reads of two half-rows, whose values are
  // neighbours in an operand, and not those of two blocks)
  uint32_t d_rd[2], a_rd[2];
#pragma unroll
  for (int p = 0; p < 2; ++p) {
    d_rd[p] = 4 * g * kWbHalf + wj * 256 + p * 128 + l32 * 4;
    a_rd[p] = kWbOperand + 4 * g * kWbHalf + wi * 256 + p * 128 + l32 * 4;
    asm("" : "+v"(d_rd[p]));
    asm("" : "+v"(a_rd[p]));
  }

  pf32x16_t acc[2][2][2];  // [16 j][16 i][real, minus imaginary]
#pragma unroll
  for (int p = 0; p < 2; ++p)
#pragma unroll
    for (int q = 0; q < 2; ++q)
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int v = 0; v < 16; ++v) acc[p][q][h][v] = 0.f;
  const bool bias_wave = db != nullptr && i0 == 0 && wi == 0;
  float bs[2][2][2] = {};  // [16 j][b][re, im] of D's entry l32 % 2

  const int nf = (rows + kWbRows - 1) / kWbRows;
#pragma unroll
  for (int f = 0; f < kWbStages - 1; ++f) {
    next_src(f);
    issue(f);
  }
  next_src(kWbStages - 1);
  auto loop = [&](auto bias_tag) __attribute__((always_inline)) {
    constexpr bool BIAS = decltype(bias_tag)::value;
    for (int f = 0; f < nf; ++f) {
      // the loads of the newer stage may stay outstanding; this wave's reads of the stage that is loaded over next have
      // returned
      asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"((kWbStages - 2) * 2 * kWbWaveRows) : "memory");
      const unsigned char* st = smem + (f % kWbStages) * kWbStage;
      uint32_t d[kWbRows / 4][2][4], a[kWbRows / 4][2][4];  // [four rows][block][half-row]
#pragma unroll
      for (int s = 0; s < kWbRows / 4; ++s)
#pragma unroll
        for (int p = 0; p < 2; ++p) {
#pragma unroll
          for (int q = 0; q < 4; ++q) d[s][p][q] = *reinterpret_cast<const uint32_t*>(st + d_rd[p] + (8 * s + q) * kWbHalf);
#pragma unroll
          for (int q = 0; q < 4; ++q) a[s][p][q] = *reinterpret_cast<const uint32_t*>(st + a_rd[p] + (8 * s + q) * kWbHalf);
        }
      issue(f + kWbStages - 1);  // over the stage read before the barrier
      next_src(f + kWbStages);
#pragma unroll
      for (int s = 0; s < kWbRows / 4; ++s) {
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          const uint32_t* w = a[s][q];
          const pbf16x8_t X = __builtin_bit_cast(pbf16x8_t, make_uint4(w[0], w[1], w[2], w[3]));
          const pbf16x8_t R = __builtin_bit_cast(
              pbf16x8_t, make_uint4(rot_conj(w[0]), rot_conj(w[1]), rot_conj(w[2]), rot_conj(w[3])));
#pragma unroll
          for (int p = 0; p < 2; ++p) {
            const pbf16x8_t Y = __builtin_bit_cast(pbf16x8_t, make_uint4(d[s][p][0], d[s][p][1], d[s][p][2], d[s][p][3]));
            acc[p][q][0] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(Y, X, acc[p][q][0], 0, 0, 0);
            acc[p][q][1] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(Y, R, acc[p][q][1], 0, 0, 0);
          }
        }
        if constexpr (BIAS) {
#pragma unroll
          for (int p = 0; p < 2; ++p)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              bs[p][q & 1][0] += bf_lo(d[s][p][q]);
              bs[p][q & 1][1] += bf_hi(d[s][p][q]);
            }
        }
      }
    }
  };
  if (bias_wave) loop(std::true_type{});
  else loop(std::false_type{});
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // the loads past the last stage write LDS too

  // lane: column i0 + 32 wi + 16 q + l32 / 2, its entry c = l32 % 2; rows j0 + 32 wj + 16 p + 4 v + 2 g + h
  const int c01 = l32 & 1;
  float* const out = n == 1 ? dW + (size_t)e * d_out * d_in * 8 : part + (size_t)plane * d_out * d_in * 8;
#pragma unroll
  for (int p = 0; p < 2; ++p)
#pragma unroll
    for (int q = 0; q < 2; ++q)
#pragma unroll
      for (int v = 0; v < 4; ++v)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int j = j0 + 32 * wj + 16 * p + 4 * v + 2 * g + h, i = i0 + 32 * wi + 16 * q + (l32 >> 1);
          const int k = 4 * v + 2 * h;
          const float4 o = half_blades(acc[p][q][0][k], -acc[p][q][1][k], acc[p][q][0][k + 1], -acc[p][q][1][k + 1], c01);
          if (j < d_out && i < d_in) *reinterpret_cast<float4*>(out + ((size_t)j * d_in + i) * 8 + 4 * c01) = o;
        }
  if (bias_wave) {
    float* const ob = n == 1 ? db + (size_t)e * d_out * 8 : dbpart + (size_t)plane * d_out * 8;
#pragma unroll
    for (int p = 0; p < 2; ++p) {
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int h = 0; h < 2; ++h) bs[p][b][h] += __shfl_xor(bs[p][b][h], 32);
      // this lane has row a = l32 % 2 of the matrix: its columns are the transposed matrix's entries, so
      // half_blades of the transpose: entries (0, a) and (1, a) there are (a, 0) and (a, 1) here
      const float4 t = half_blades(bs[p][0][0], bs[p][0][1], bs[p][1][0], bs[p][1][1], c01);
      const int j = j0 + 32 * wj + 16 * p + (l32 >> 1);
      // transposing keeps every blade but v2 and b13 (the antisymmetric ones), which change sign
      const float4 o = c01 ? make_float4(t.x, -t.y, t.z, t.w) : make_float4(t.x, t.y, -t.z, t.w);
      if (g == 0 && j < d_out) *reinterpret_cast<float4*>(ob + (size_t)j * 8 + 4 * c01) = o;
    }
  }
}

// dW and db of the experts whose rows are several chunks, their planes added in order.
// A thread per four values, blockIdx.y the expert.
__global__ __launch_bounds__(256) void weight_grad_bf16_reduce_kernel(const float* __restrict__ part,
                                                                      const float* __restrict__ dbpart,
                                                                      const int32_t* __restrict__ offsets, int P, int limit,
                                                                      int E, int d_in, int d_out,
                                                                      float* __restrict__ dW, float* __restrict__ db) {
  const int e = blockIdx.y, lane = threadIdx.x & 63;
  const WbExpert x = wb_experts(offsets, E, P, limit, lane);
  const int n = __builtin_amdgcn_readlane(x.n, e);
  if (n <= 1) return;
  const int first = __builtin_amdgcn_readlane(wave_scan<false>(x.n > 1 ? x.n : 0), e) - n;
  const size_t nw = (size_t)d_out * d_in * 2, nb = db != nullptr ? (size_t)d_out * 2 : 0;
  size_t u = (size_t)blockIdx.x * 256 + threadIdx.x;
  if (u >= nw + nb) return;
  const bool bias = u >= nw;
  const size_t stride = bias ? nb : nw;
  if (bias) u -= nw;
  const float4* p = reinterpret_cast<const float4*>(bias ? dbpart : part) + (size_t)first * stride + u;
  float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
  for (int q = 0; q < n; ++q) {
    const float4 v = p[(size_t)q * stride];
    s.x += v.x; s.y += v.y; s.z += v.z; s.w += v.w;
  }
  (reinterpret_cast<float4*>(bias ? db : dW) + (size_t)e * stride)[u] = s;
}

long long wb_tiles(int d_in, int d_out) {
  return (long long)((d_out + kWbTile - 1) / kWbTile) * ((d_in + kWbTile - 1) / kWbTile);
}
// The rows of a chunk at most: what each of the 512 workgroups that the chip holds would have of all rows' tiles,
// within limits.  More rows leave CUs idle at the end, fewer make more planes, which the reduction reads at the
// rate of memory: 8192 tokens, d = 128, F = 512, E = 32, k = 4, Zipf's law take 171 us with at most 512 rows, 158 with
// 768, 153 with this rule's 1024; 1500 tokens, d = 100, F = 300, E = 12, k = 3 take 33 us with at least 512 rows, 27 with
// 256, 29 with 128.
//
// Few rows take one chunk an expert, no planes and no second launch.  That pays while the largest expert has little
// more than the 252 rows of the shortest chunks, which the host does not know: it is taken for Zipf's law over E experts
// (exponent 1.2), whose crossover lies at or above 252 + 96 log2(E) rows at all widths measured.  One chunk and chunks of
// 252, us by graph replay, d = 64, F = 256: E = 1, 256 rows 18.8 and 15.3, 516 rows 30.4 and 18.6; E = 4, 400 rows 16.6
// and 18.2, 516 rows 19.4 and 15.7; E = 8, 516 rows 17.4 and 19.0, 640 rows 19.5 and 15.8; E = 16, 640 rows 18.4 and
// 20.3, 768 rows 20.6 and 17.0; E = 32, 768 rows 20.0 and 22.4, 900 rows 22.1 and 18.9; E = 64, 768 rows 20.6 and 24.7,
// 900 rows 22.2 and 21.6 (d = 256, F = 1024: E = 4, 400 rows 25.8 and 29.8, 516 rows 30.3 and 29.1; E = 32, 768 rows 82 and
// 107).  Even experts gain at every such size (E = 8, 516 rows 10.3 and 11.9); all rows at one of eight experts lose
// (516 rows 30.6 and 18.2).
int rows_of_one_chunk(int E) {
  int log2e = 0;
  while (E >> (log2e + 1)) ++log2e;
  return 252 + 96 * log2e;
}
int chunk_rows(int P, int E, int d_in, int d_out) {
  const int few = rows_of_one_chunk(E);
  static_assert((252 + 96 * 6) <= kWbMaxChunk && 252 % kWbRows == 0 && 96 % kWbRows == 0, "chunks are whole stages");
  if (P <= few) return few;
  const long long even = (long long)P * wb_tiles(d_in, d_out) / 512;
  return (int)std::min<long long>(kWbMaxChunk, std::max<long long>(kWbMinChunk, even)) / kWbRows * kWbRows;
}
// chunks there can be with the experts without any, and planes of the experts that have several: such an expert
// has more than `limit` rows
long long wb_chunks(long long P, int E, int limit) { return P / limit + E; }
long long wb_planes(long long P, int E, int limit) {
  return P > limit ? P / limit + std::min<long long>(E, P / (limit + 1)) : 0;
}

}  // namespace

const char* weight_grad_bf16_limit(int P_max, int E, int d_in, int d_out, bool gathered, int a_rows) {
  // offsets inside a chunk, past its end by the stages in flight, are 32 bits with one bit for "outside"
  if ((long long)(kWbMaxChunk + kWbRows * (kWbStages + 1)) * std::max(d_in, d_out) * 16 >= 1LL << 31)
    return "the weight gradient's chunks of rows reach 2 GiB";
  if ((wb_chunks(P_max, E, chunk_rows(P_max, E, d_in, d_out)) + 8) * wb_tiles(d_in, d_out) >= 1LL << 24)
    return "the weight gradient exceeds a launch";
  if (gathered && (long long)a_rows * d_in * 16 >= 1LL << 31) return "gathered rows span 2 GiB or more";
  return nullptr;
}

size_t weight_grad_bf16_workspace_bytes(int P_max, int E, int d_in, int d_out) {
  return (size_t)wb_planes(P_max, E, chunk_rows(P_max, E, d_in, d_out)) * d_out * (d_in + 1) * 8 * sizeof(float);
}

int weight_grad_bf16(const void* dy, const void* a, int a_rows, const int32_t* gather, const int32_t* offsets, int P_max,
                     int E, int d_in, int d_out, float* dW, float* db, void* workspace, hipStream_t stream) {
  if (E == 0) return 0;
  const int limit = chunk_rows(P_max, E, d_in, d_out);
  const long long planes = wb_planes(P_max, E, limit), chunks = wb_chunks(P_max, E, limit);
  float* part = static_cast<float*>(workspace);
  float* dbpart = part + (size_t)planes * d_out * d_in * 8;
  const int n_xcd = 8;  // workgroups go to the XCDs round robin (8 on MI355X)
  const long long nt = wb_tiles(d_in, d_out);
  const dim3 grid((unsigned)((chunks + n_xcd - 1) / n_xcd * n_xcd * nt));
  auto* kernel = gather ? weight_grad_bf16_kernel<true> : weight_grad_bf16_kernel<false>;
  hipLaunchKernelGGL(kernel, grid, dim3(256), 0, stream, static_cast<const uint16_t*>(dy), static_cast<const uint16_t*>(a),
                     a_rows, gather, offsets, P_max, limit, E, d_in, d_out, n_xcd, part, dbpart, dW, db);
  if (check_launch("weight gradient (bf16)")) return -1;
  if (planes == 0) return 0;
  const size_t n4 = (size_t)d_out * (d_in + (db ? 1 : 0)) * 2;
  hipLaunchKernelGGL(weight_grad_bf16_reduce_kernel, dim3((unsigned)((n4 + 255) / 256), E), dim3(256), 0, stream, part,
                     dbpart, offsets, P_max, limit, E, d_in, d_out, dW, db);
  return check_launch("weight gradient (bf16, reduction)");
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
  const char* why = weight_grad_bf16_limit(P_max, E, d_in, d_out, gather != nullptr, a_rows);
  YGG_CHECK_ARG(!why, "ygg_grouped_weight_grad_pauli_bf16: %s (P_max=%d d_in=%d d_out=%d a_rows=%d)", why, P_max, d_in, d_out,
                a_rows);
  if (E == 0) return 0;
  YGG_CHECK_ARG(offsets && dW && (P_max == 0 || (dy_pauli && a_pauli)),
                "ygg_grouped_weight_grad_pauli_bf16: null pointer argument");
  const size_t need = weight_grad_bf16_workspace_bytes(P_max, E, d_in, d_out);
  YGG_CHECK_ARG(need == 0 || (workspace && workspace_bytes >= need),
                "ygg_grouped_weight_grad_pauli_bf16: workspace of %zu bytes, need %zu", workspace ? workspace_bytes : 0,
                need);
  return weight_grad_bf16(dy_pauli, a_pauli, a_rows, gather, offsets, P_max, E, d_in, d_out, dW, db, workspace, stream);
}
