// int8_rows.hip -- expert products of int8 rows with int8 weights (CliffordLinear, clifford_linear.py:84-123, of every
// expert's rows; the reference has no int8 product).
//
// A geometric product is a product of complex 2x2 matrices, Y_j = sum_i W_ji X_i.  With the entries of W as codes of one
// scale an output channel and those of X / 2 as codes of one scale a row, the sums run in 32-bit integers and are exact:
//   Re Y = sum U xr - V xi,  Im Y = sum U xi + V xr,  Y = s_w s_x (that),
// 32 multiply-adds a pair of multivectors.  The halves make the way back to blades plain sums.
//
// Quantization of a row: a its largest entry, at least 2^-100; s = a / 127; q = rint(e (127 / a)), each operation
// rounded to fp32 -- |q| <= 127, as e (127 / a) <= 127 (1 + 2^-23).  A row with an infinity or a NaN gets the
// scale NaN, and so its outputs are NaN; a row of zeros has codes 0 and gives the bias.

#include <hip/hip_runtime.h>

#include <algorithm>

#include "int8_rows.h"
#include "rows.h"
#include "ygg_common.h"

namespace ygg {
namespace {

constexpr float kI8Tiny = 0x1p-100f;

__device__ __forceinline__ void half_entries(const float v[8], float e[8]) {  // [b][c][re, im]
  float h[8];
#pragma unroll
  for (int q = 0; q < 8; ++q) h[q] = 0.5f * v[q];
  blade_to_pauli(h, e, e + 4);
}
// the codes of a multivector's four (b, part) pairs, each (c0, c1) as 16 bits
__device__ __forceinline__ void codes_of(const float v[8], float inv, uint32_t q[4]) {
  float e[8];
  half_entries(v, e);
#pragma unroll
  for (int b = 0; b < 2; ++b)
#pragma unroll
    for (int part = 0; part < 2; ++part) {
      const int c0 = (int)rintf(e[4 * b + part] * inv), c1 = (int)rintf(e[4 * b + 2 + part] * inv);
      q[2 * b + part] = (uint32_t)(c0 & 0xff) | (uint32_t)(c1 & 0xff) << 8;
    }
}

// Lane exchanges within rows of 16 lanes, on the vector units (through LDS the sums and codes of a row of 128 multivectors
// took a third longer).
template <int CTRL>
__device__ __forceinline__ uint32_t dpp(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_mov_dpp((int)v, CTRL, 0xf, 0xf, true);
}
constexpr int kXor1 = 0xB1, kXor2 = 0x4E, kHalfMirror = 0x141, kMirror = 0x140;
__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
  v = max(v, dpp<kXor1>(v));
  v = max(v, dpp<kXor2>(v));
  v = max(v, dpp<kHalfMirror>(v));
  v = max(v, dpp<kMirror>(v));
  const uint32_t a = __builtin_amdgcn_readlane((int)v, 0), b = __builtin_amdgcn_readlane((int)v, 16);
  const uint32_t c = __builtin_amdgcn_readlane((int)v, 32), d = __builtin_amdgcn_readlane((int)v, 48);
  return max(max(a, b), max(c, d));
}

// WAVES waves a row, four waves a workgroup; a lane takes every 64 WAVES-th multivector, KEEP of them kept from the pass
// that finds the largest entry to the one that writes the codes.
template <typename T, int WAVES, int KEEP>
__global__ __launch_bounds__(256) void quantize_rows_kernel(const T* __restrict__ x, int rows, int d,
                                                            unsigned char* __restrict__ codes, float* __restrict__ scale) {
  constexpr int RPB = 4 / WAVES;
  __shared__ uint32_t s_max[4];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int row = blockIdx.x * RPB + wave / WAVES;
  if (WAVES == 1 && row >= rows) return;  // (with several waves a row, every workgroup has one)
  const int first = (wave % WAVES) * 64 + lane;
  constexpr int STRIDE = 64 * WAVES;
  RawMv<T> kept[KEEP];
  uint32_t top = 0;
  auto look = [&](const RawMv<T>& m) {
    float v[8], e[8];
    unpack(m, v);
    half_entries(v, e);
#pragma unroll
    for (int q = 0; q < 8; ++q) top = max(top, __builtin_bit_cast(uint32_t, e[q]) & 0x7fffffffu);  // NaN above infinity
  };
#pragma unroll
  for (int u = 0; u < KEEP; ++u)
    if (first + u * STRIDE < d) kept[u] = load_raw(x, (size_t)row * d + first + u * STRIDE);
#pragma unroll
  for (int u = 0; u < KEEP; ++u)
    if (first + u * STRIDE < d) look(kept[u]);
  for (int i = first + KEEP * STRIDE; i < d; i += STRIDE) look(load_raw(x, (size_t)row * d + i));
  top = wave_max(top);
  if constexpr (WAVES > 1) {
    if (lane == 0) s_max[wave] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < WAVES; ++w) top = max(top, s_max[w]);
  }
  const bool finite = top < 0x7f800000u;
  const float a = fmaxf(__builtin_bit_cast(float, finite ? top : 0u), kI8Tiny);
  const float inv = 127.0f / a;
  if (first == 0) scale[row] = finite ? a / 127.0f : __builtin_nanf("");
  const int steps = i8_steps(d);
  unsigned char* const out = codes + (size_t)row * i8_row_bytes(d);
  auto write = [&](int i, const float v[8]) {
    // four lanes hold four inputs' (b, part) pairs; the exchange gives lane p of them pair p of all four: 8 bytes
    uint32_t q[4];
    codes_of(v, finite ? inv : 0.f, q);
    const uint32_t w0 = q[0] | q[1] << 16, w1 = q[2] | q[3] << 16;
    const bool odd = lane & 1, up = lane & 2;
    const uint32_t o0 = dpp<kXor1>(w0), o1 = dpp<kXor1>(w1);
    const uint32_t p0 = odd ? (o0 >> 16 | (w0 & 0xffff0000u)) : (w0 & 0xffffu) | o0 << 16;  // pairs 0 and 1 of two inputs
    const uint32_t p1 = odd ? (o1 >> 16 | (w1 & 0xffff0000u)) : (w1 & 0xffffu) | o1 << 16;  // pairs 2 and 3
    const uint32_t r0 = dpp<kXor2>(p0), r1 = dpp<kXor2>(p1);
    const uint2 eight = up ? make_uint2(r1, p1) : make_uint2(p0, r0);
    const int pair = lane & 3;  // 2 b + part
    const int ks = i >> 5, g = (i >> 3) & 3, half = (i >> 2) & 1;
    *reinterpret_cast<uint2*>(out + (size_t)((pair >> 1) * steps + ks) * kI8StepBytes + (pair & 1) * 64 + g * 16 + half * 8) =
        eight;
  };
  const int end = steps * kI8Step;  // (whole groups of 32 lanes write)
#pragma unroll
  for (int u = 0; u < KEEP; ++u) {
    const int i = first + u * STRIDE;
    if (i >= end) break;
    float v[8] = {};
    if (i < d) unpack(kept[u], v);
    write(i, v);
  }
  for (int i = first + KEEP * STRIDE; i < end; i += STRIDE) {
    float v[8] = {};
    if (i < d) load_mv(x, (size_t)row * d + i, v);
    write(i, v);
  }
}

template <typename T>
void launch_quantize(const void* x, int rows, int d, void* codes, float* scale, hipStream_t stream) {
  const T* X = static_cast<const T*>(x);
  unsigned char* C = static_cast<unsigned char*>(codes);
  const unsigned quarter = (unsigned)(((long long)rows + 3) / 4);
  if (d <= 64)
    quantize_rows_kernel<T, 1, 1><<<quarter, 256, 0, stream>>>(X, rows, d, C, scale);
  else if (d <= 256)
    quantize_rows_kernel<T, 1, 4><<<quarter, 256, 0, stream>>>(X, rows, d, C, scale);
  else
    quantize_rows_kernel<T, 4, 4><<<(unsigned)rows, 256, 0, stream>>>(X, rows, d, C, scale);
}

// ---- the product -------------------------------------------------------------------

// sums of four byte products
__device__ __forceinline__ int dot4(uint32_t a, uint32_t b, int c) { return __builtin_amdgcn_sdot4((int)a, (int)b, c, false); }

__device__ __forceinline__ void store_out(float* y, size_t n, const float v[8]) { store_mv(y, n, v); }
__device__ __forceinline__ void store_out(uint16_t* y, size_t n, const float v[8]) { store_mv(y, n, v); }

// A thread per output multivector, four-byte products on the vector units.
template <int ACT, typename TY>
__global__ __launch_bounds__(256) void int8_linear_simple_kernel(const uint4* __restrict__ X, const float* __restrict__ xs,
                                                                 int x_rows, const int32_t* __restrict__ gather,
                                                                 const uint4* __restrict__ W, const float* __restrict__ ws,
                                                                 const float* __restrict__ bias,
                                                                 const int32_t* __restrict__ offsets, int E, int d_in,
                                                                 int d_out, int P_max, TY* __restrict__ y) {
  const int r = blockIdx.x;
  const int j = blockIdx.y * 256 + threadIdx.x;
  if (r >= min(offsets[E], P_max) || j >= d_out) return;
  int e = 0;
  while (offsets[e + 1] <= r) ++e;
  const int src = gather ? gather[r] : r;
  const int steps = i8_steps(d_in);
  const bool in = (unsigned)src < (unsigned)x_rows;  // (else a row of zeros)
  const uint4* xr = X + (size_t)(in ? src : 0) * steps * 16;
  const uint4* w = W + (size_t)e * (i8_expert_bytes(d_out, d_in) / 16) + (size_t)(j >> 3) * steps * 128 + 2 * (j & 7);
  int re[2][2] = {}, im[2][2] = {};  // [a][b]
  auto dot = [](const uint4& p, const uint4& q, int c) {
    return dot4(p.x, q.x, dot4(p.y, q.y, dot4(p.z, q.z, dot4(p.w, q.w, c))));
  };
  for (int ks = 0; ks < steps; ++ks)
    for (int g = 0; g < 4; ++g)
      for (int a = 0; a < 2; ++a) {
        const uint4 U = w[(size_t)ks * 128 + g * 16 + a], V = w[(size_t)ks * 128 + 64 + g * 16 + a];
        for (int b = 0; b < 2; ++b) {
          const uint4 xre = xr[(size_t)(b * steps + ks) * 8 + g], xim = xr[(size_t)(b * steps + ks) * 8 + 4 + g];
          re[a][b] = dot(U, xre, re[a][b]) - dot(V, xim, 0);
          im[a][b] = dot(U, xim, dot(V, xre, im[a][b]));
        }
      }
  float o[8], bv[8] = {};
  if (bias) {
#pragma unroll
    for (int c = 0; c < 8; ++c) bv[c] = bias[((size_t)e * d_out + j) * 8 + blade_to_mask(c)];
  }
  i8_blades(re[0][0], im[0][0], re[0][1], im[0][1], re[1][0], im[1][0], re[1][1], im[1][1],
            ws[(size_t)e * d_out + j] * (in ? xs[src] : 0.f), bv, o);
  activate_blade<ACT>(o);
  store_out(y, (size_t)r * d_out + j, o);
}

template <int ACT, typename TY>
int launch_linear(const void* x, const float* xs, int x_rows, const int32_t* gather, int P, const void* w, const float* ws,
                  const float* bias, const int32_t* offsets, int E, int d_in, int d_out, void* y, hipStream_t stream) {
  int8_linear_simple_kernel<ACT, TY><<<dim3((unsigned)P, (unsigned)((d_out + 255) / 256)), 256, 0, stream>>>(
      static_cast<const uint4*>(x), xs, x_rows, gather, static_cast<const uint4*>(w), ws, bias, offsets, E, d_in, d_out, P,
      static_cast<TY*>(y));
  return check_launch("int8_grouped_linear");
}

}  // namespace

size_t int8_rows_bytes(size_t rows, int d) { return rows * i8_row_bytes(d); }

const char* int8_linear_limit(int x_rows, bool gathered, int E, int d_in, int d_out) {
  if (d_in > kI8MaxInputs) return "int8 products sum at most 16384 inputs in 32 bits";
  if (d_out > 1 << 19) return "int8 products write at most 524288 channels";
  if (i8_expert_bytes(d_out, d_in) >= 0x7fffffffull) return "one expert's int8 weights exceed 2 GiB";
  if (gathered && (uint64_t)x_rows * i8_row_bytes(d_in) >= 0x7fffffffull) return "the gathered int8 rows exceed 2 GiB";
  return nullptr;
}

}  // namespace ygg

using namespace ygg;

YGG_API size_t ygg_int8_rows_bytes(int rows, int d) { return rows < 0 || d < 1 ? 0 : int8_rows_bytes((size_t)rows, d); }

YGG_API int ygg_quantize_rows(const void* x, int x_dtype, int rows, int d, void* codes, float* scale, hipStream_t stream) {
  YGG_CHECK_ARG(rows >= 0 && d >= 1, "ygg_quantize_rows: bad sizes rows=%d d=%d", rows, d);
  YGG_CHECK_ARG(x_dtype == kF32 || x_dtype == kBF16, "ygg_quantize_rows: dtype %d unsupported", x_dtype);
  if (rows == 0) return 0;
  YGG_CHECK_ARG(x && codes && scale, "ygg_quantize_rows: null pointer");
  const size_t xb = (size_t)rows * d * 8 * dtype_size(x_dtype), cb = int8_rows_bytes((size_t)rows, d);
  YGG_CHECK_ARG(!overlap(x, xb, codes, cb) && !overlap(x, xb, scale, (size_t)rows * 4) &&
                    !overlap(codes, cb, scale, (size_t)rows * 4),
                "ygg_quantize_rows: x, codes and scale must not share memory");
  if (x_dtype == kF32) launch_quantize<float>(x, rows, d, codes, scale, stream);
  else launch_quantize<uint16_t>(x, rows, d, codes, scale, stream);
  return check_launch("quantize_rows");
}

YGG_API int ygg_int8_grouped_linear(const void* codes, const float* x_scale, int x_rows, const int32_t* gather, int P_max,
                                    const void* w_prepared, const float* w_scale, const float* bias, const int32_t* offsets,
                                    int E, int d_in, int d_out, int act, void* y, int y_dtype, hipStream_t stream) {
  YGG_CHECK_ARG(x_rows >= 0 && P_max >= 0 && E >= 1 && E <= 64 && d_in >= 1 && d_in <= kI8MaxInputs && d_out >= 1,
                "ygg_int8_grouped_linear: bad sizes x_rows=%d P_max=%d E=%d d_in=%d d_out=%d (E <= 64, d_in <= %d)", x_rows,
                P_max, E, d_in, d_out, kI8MaxInputs);
  YGG_CHECK_ARG(act >= kActNone && act <= kActSigmoid, "ygg_int8_grouped_linear: activation %d", act);
  YGG_CHECK_ARG(y_dtype == kF32 || y_dtype == kBF16, "ygg_int8_grouped_linear: output dtype %d unsupported", y_dtype);
  const char* const why = int8_linear_limit(x_rows, gather != nullptr, E, d_in, d_out);
  YGG_CHECK_ARG(!why, "ygg_int8_grouped_linear: %s (x_rows=%d E=%d d_in=%d d_out=%d)", why, x_rows, E, d_in, d_out);
  if (P_max == 0) return 0;
  YGG_CHECK_ARG(codes && x_scale && w_prepared && w_scale && offsets && y, "ygg_int8_grouped_linear: null pointer");
  YGG_CHECK_ARG(gather || x_rows >= P_max, "ygg_int8_grouped_linear: %d rows of x for %d product rows", x_rows, P_max);
  // few rows: the weights set the time (32 rows of 64 experts, 256 -> 1024: 18.7 us, 21.5 on the tiles; 4500 rows of 12,
  // 100 -> 300: 77 us, 25 on the tiles)
  if (P_max > 64)
    return int8_tile_linear(codes, x_scale, x_rows, gather, P_max, w_prepared, w_scale, bias, offsets, E, d_in, d_out, act, y,
                            y_dtype, stream);
#define YGG_I8(A)                                                                                                           \
  return y_dtype == kF32 ? launch_linear<A, float>(codes, x_scale, x_rows, gather, P_max, w_prepared, w_scale, bias,       \
                                                   offsets, E, d_in, d_out, y, stream)                                     \
                         : launch_linear<A, uint16_t>(codes, x_scale, x_rows, gather, P_max, w_prepared, w_scale, bias,    \
                                                      offsets, E, d_in, d_out, y, stream)
  switch (act) {
    case kActNone: YGG_I8(kActNone);
    case kActGelu: YGG_I8(kActGelu);
    case kActRelu: YGG_I8(kActRelu);
    default: YGG_I8(kActSigmoid);
  }
#undef YGG_I8
}
