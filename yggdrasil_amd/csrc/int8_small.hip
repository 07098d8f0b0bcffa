// int8_small.hip -- the product of int8 rows with int8 weights (int8_rows.hip: the mathematics; int8_tile.hip: the same for
// enough rows) for few rows, where the weights are read once or a few times and set the time.
//
// A wave is a workgroup: 8 tokens x 16 channels on v_mfma_i32_16x16x64_i8, whose K of 64 is the real or the imaginary
// part of a K step of 32 inputs; Re and Im as in int8_tile.hip.  Nothing is shared, so there is no barrier: operands
// come straight to registers, kRing steps of them on their way, the weights asked for before the rows' places are
// known.  The sums are whole numbers and the epilogue is the tiles', so a row's outputs are the same bit for bit.
// Bound by the weight stream (32 rows of 64 experts, 256 -> 1024: 12.7 us, about 50 MB at 4 TB/s) and, where that is
// short, by the chain of dependent loads in front of it: bounds, places, rows (512 rows of 8 experts, 64 -> 256: 5.5 us).
// 16 or 32 tokens a wave took longer wherever this kernel is taken (13.8 and 14.7 us, 6.0 and 6.6).

#include <hip/hip_runtime.h>

#include <algorithm>

#include "int8_rows.h"
#include "rows.h"
#include "ygg_common.h"

namespace ygg {
namespace {

typedef int i32x4_t __attribute__((ext_vector_type(4)));
constexpr int kTokens = 8, kRing = 4;

template <int ACT, typename TY>
__global__ __launch_bounds__(64) void int8_small_kernel(const unsigned char* __restrict__ X, uint64_t x_bytes,
                                                        const float* __restrict__ xs, int x_rows,
                                                        const int32_t* __restrict__ gather,
                                                        const unsigned char* __restrict__ W, const float* __restrict__ ws,
                                                        const float* __restrict__ bias, const int32_t* __restrict__ offsets,
                                                        int E, int d_in, int d_out, int P_max, TY* __restrict__ y) {
  const int lane = threadIdx.x, l16 = lane & 15, g = lane >> 4;
  const int n_ct = (d_out + 15) / 16;
  const int ct = blockIdx.x % n_ct, rt = blockIdx.x / n_ct;
  // lane e: expert e's rows; a scan finds the one that holds row tile rt
  auto inside = [&](int at) { return lane < E ? min(max(offsets[lane + at], 0), P_max) : 0; };
  const int v_beg = inside(0), v_end = max(inside(1), v_beg);
  const int v_nt = (v_end - v_beg + kTokens - 1) / kTokens;
  int incl = v_nt;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int p = __shfl_up(incl, o);
    if (lane >= o) incl += p;
  }
  const uint64_t after = __ballot(incl > rt);
  if (after == 0) return;
  const int e = (int)__builtin_ctzll(after);
  const int row0 = __builtin_amdgcn_readlane(v_beg, e) +
                   (rt - (__builtin_amdgcn_readlane(incl, e) - __builtin_amdgcn_readlane(v_nt, e))) * kTokens;
  const int rows = min(kTokens, __builtin_amdgcn_readlane(v_end, e) - row0);

  const int steps = i8_steps(d_in);
  const uint32_t half_bytes = (uint32_t)steps * kI8StepBytes;
  auto rsrc_from = [](const void* base, uint64_t off, uint64_t bytes) __attribute__((always_inline)) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(static_cast<const char*>(base)) + off, (short)0,
                                             (uint32_t)(bytes < 0x7fffffffull ? bytes : 0x7fffffffull), kBufferFlags);
  };
  const size_t expert_bytes = i8_expert_bytes(d_out, d_in);
  const uint64_t first = gather ? 0 : (uint64_t)row0 * half_bytes * 2;
  const __amdgpu_buffer_rsrc_t x_rsrc = rsrc_from(X, first, x_bytes - first);
  const __amdgpu_buffer_rsrc_t w_rsrc = rsrc_from(W, (uint64_t)e * expert_bytes, expert_bytes);
  // the rows of this lane's operands (half-row l16) and outputs (2 g, 2 g + 1); past the tile's end, and for a gathered
  // place outside x, zeros
  auto source = [&](int tok) { return tok >= rows ? -1 : gather ? gather[row0 + tok] : tok; };
  const int a_src = source(l16 >> 1), o_src[2] = {source(2 * g), source(2 * g + 1)};
  // (a block of channels behind the last lies past the expert's weights: zeros)
  const uint32_t w_off = (uint32_t)(2 * ct + (l16 >> 3)) * steps * kI8BlockBytes + g * 256 + (l16 & 7) * 32;
  i32x4_t xr[kRing], xi[kRing], u[kRing][2], v[kRing][2];
  auto load = [&](__amdgpu_buffer_rsrc_t r, uint32_t off) {
    return __builtin_bit_cast(i32x4_t, __builtin_amdgcn_raw_buffer_load_b128(r, off, 0, 0));
  };
  auto load_w = [&](int slot, int ks) __attribute__((always_inline)) {
    const uint32_t off = ks < steps ? w_off + (uint32_t)ks * kI8BlockBytes : kBufferOff;
#pragma unroll
    for (int a = 0; a < 2; ++a) {
      u[slot][a] = load(w_rsrc, off + a * 16);
      v[slot][a] = load(w_rsrc, off + a * 16 + 1024);
    }
  };
#pragma unroll
  for (int k = 0; k < kRing; ++k) load_w(k, k);
  const int j = ct * 16 + l16;
  const size_t ej = (size_t)e * d_out + min(j, d_out - 1);
  const float sw = ws[ej];
  const __amdgpu_buffer_rsrc_t b_rsrc = rsrc_from(bias, 0, bias ? (uint64_t)E * d_out * 32 : 0);
  const i32x4_t lo = load(b_rsrc, (uint32_t)ej * 32), hi = load(b_rsrc, (uint32_t)ej * 32 + 16);
  float bv[8];
#pragma unroll
  for (int c = 0; c < 8; ++c) {
    const int m = blade_to_mask(c);
    bv[c] = __builtin_bit_cast(float, m < 4 ? lo[m] : hi[m - 4]);
  }
  float sx[2];
#pragma unroll
  for (int h = 0; h < 2; ++h)
    sx[h] = (unsigned)o_src[h] < (unsigned)x_rows ? xs[(gather ? 0 : row0) + (size_t)o_src[h]] : 0.f;
  const uint32_t a_off =
      (unsigned)a_src < (unsigned)x_rows ? (uint32_t)(2 * a_src + (l16 & 1)) * half_bytes + g * 16 : kBufferOff;
  auto load_x = [&](int slot, int ks) __attribute__((always_inline)) {
    const uint32_t off = ks < steps ? a_off + (uint32_t)ks * kI8StepBytes : kBufferOff;
    xr[slot] = load(x_rsrc, off);
    xi[slot] = load(x_rsrc, off + 64);
  };
#pragma unroll
  for (int k = 0; k < kRing; ++k) load_x(k, k);

  i32x4_t acc[2][2] = {};  // [a][re, im]
  int vsum[2] = {};
#pragma unroll 1
  for (int k0 = 0; k0 < steps; k0 += kRing) {
#pragma unroll
    for (int q = 0; q < kRing; ++q) {
#pragma unroll
      for (int a = 0; a < 2; ++a) {
        acc[a][0] = __builtin_amdgcn_mfma_i32_16x16x64_i8(xr[q], u[q][a], acc[a][0], 0, 0, 0);
        acc[a][1] = __builtin_amdgcn_mfma_i32_16x16x64_i8(xi[q], u[q][a], acc[a][1], 0, 0, 0);
        acc[a][0] = __builtin_amdgcn_mfma_i32_16x16x64_i8(~xi[q], v[q][a], acc[a][0], 0, 0, 0);
        acc[a][1] = __builtin_amdgcn_mfma_i32_16x16x64_i8(xr[q], v[q][a], acc[a][1], 0, 0, 0);
#pragma unroll
        for (int c = 0; c < 4; ++c) vsum[a] = __builtin_amdgcn_sdot4(v[q][a][c], 0x01010101, vsum[a], false);
      }
      // (past the last step: zeros, without traffic; their products add nothing)
      load_w(q, k0 + q + kRing);
      load_x(q, k0 + q + kRing);
    }
  }
#pragma unroll
  for (int a = 0; a < 2; ++a) {
    vsum[a] += __shfl_xor(vsum[a], 16);
    vsum[a] += __shfl_xor(vsum[a], 32);
  }
  if (j >= d_out) return;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int tok = 2 * g + h;  // its halves b = 0, 1 are sums 2 h, 2 h + 1
    if (tok >= rows) continue;
    float o[8];
    i8_blades(acc[0][0][2 * h] + vsum[0], acc[0][1][2 * h], acc[0][0][2 * h + 1] + vsum[0], acc[0][1][2 * h + 1],
              acc[1][0][2 * h] + vsum[1], acc[1][1][2 * h], acc[1][0][2 * h + 1] + vsum[1], acc[1][1][2 * h + 1], sw * sx[h], bv,
              o);
    activate_blade<ACT>(o);
    store_mv(y, (size_t)(row0 + tok) * d_out + j, o);
  }
}

template <int ACT, typename TY>
int launch_small(const void* x, const float* xs, int x_rows, const int32_t* gather, int P, const void* w, const float* ws,
                 const float* bias, const int32_t* offsets, int E, int d_in, int d_out, void* y, hipStream_t stream) {
  // at most this many tiles of rows, whatever the experts' shares
  const long long tiles = std::min<long long>(P, P / kTokens + E);
  int8_small_kernel<ACT, TY><<<(unsigned)(tiles * ((d_out + 15) / 16)), 64, 0, stream>>>(
      static_cast<const unsigned char*>(x), (uint64_t)x_rows * i8_row_bytes(d_in), xs, x_rows, gather,
      static_cast<const unsigned char*>(w), ws, bias, offsets, E, d_in, d_out, P, static_cast<TY*>(y));
  return check_launch("int8_small");
}

}  // namespace

// Few outputs, counted as this kernel computes them (channels in groups of 16): the tiles, 64 x 64, leave most of the chip
// idle.  A product, few rows / tiles, us: 8 rows, E = 32, 128 -> 512: 4.1 / 8.6; 32, E = 64, 256 -> 1024: 12.7 / 16.9,
// 1024 -> 256: 13.6 / 26.1; 512, E = 8, 256 -> 64: 5.3 / 9.9; 1024, E = 32, 512 -> 128: 13.1 / 15.9, 128 -> 512: 15.8 / 11.5;
// 2048, E = 8, 256 -> 64: 7.8 / 10.1, 64 -> 256: 11.8 / 8.8; 300, E = 4, 256 -> 1024: 12.9 / 12.0; 2048, E = 32, 512 -> 128:
// 19.9 / 16.4.  One expert, where rows are most: 3125 rows, 512 -> 64: 15.0 / 18.0, 6250: 25.7 / 19.0.  Narrow outputs (the
// call's host time hides what is below 8): 12500 rows to 1, 4 or 16 channels of 512 inputs 14.6 to 15 / 19; 25000 rows,
// 32 inputs 8.8 to 9.5 / 8.3, 128: 10.5 / 11.2, 512: 25 / 27; 100000 rows to 1 or 4 channels, 32 inputs 24 / 16.4, 128: 29.7 / 28.7,
// 512: 92 to 96 / 92 to 93.
bool int8_small_pays(int P, int d_out) { return (long long)P * ((d_out + 15LL) / 16 * 16) <= 200000; }

int int8_small_linear(const void* x, const float* xs, int x_rows, const int32_t* gather, int P, const void* w,
                      const float* ws, const float* bias, const int32_t* offsets, int E, int d_in, int d_out, int act,
                      void* y, int y_dtype, hipStream_t stream) {
#define YGG_I8(A)                                                                                                             \
  return y_dtype == kF32 ? launch_small<A, float>(x, xs, x_rows, gather, P, w, ws, bias, offsets, E, d_in, d_out, y, stream)  \
                         : launch_small<A, uint16_t>(x, xs, x_rows, gather, P, w, ws, bias, offsets, E, d_in, d_out, y, stream)
  switch (act) {
    case kActNone: YGG_I8(kActNone);
    case kActGelu: YGG_I8(kActGelu);
    case kActRelu: YGG_I8(kActRelu);
    default: YGG_I8(kActSigmoid);
  }
#undef YGG_I8
}

}  // namespace ygg
