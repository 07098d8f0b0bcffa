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

// Bounds of experts' ranges as a caller has them, indexes of 4 or 8 bytes: brought into [0, P] and into ascending order,
// by one wave.
struct Ranges {
  const void *offsets = nullptr, *counts = nullptr;
  int index_bytes = 4, E = 0, P = 0;
  int32_t* bounds = nullptr;
};
template <typename I>
__device__ __forceinline__ void write_bounds(const Ranges& r) {
  const int lane = threadIdx.x & 63;
  const long long at = lane < r.E ? static_cast<const I*>(r.offsets)[lane] : 0;
  const long long count = lane < r.E ? static_cast<const I*>(r.counts)[lane] : 0;
  long long end;  // (a sum past 64 bits has the sign of its terms)
  if (__builtin_add_overflow(at, count, &end)) end = at < 0 ? at : r.P;
  auto clip = [&](long long v) { return (int)min(max(v, 0LL), (long long)r.P); };
  int v = lane < r.E ? clip(at) : 0;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int p = __shfl_up(v, o);
    if (lane >= o) v = max(v, p);
  }
  if (lane < r.E) r.bounds[lane] = v;
  if (lane == r.E - 1) r.bounds[r.E] = max(v, clip(end));
}
__device__ __forceinline__ void write_ranges(const Ranges& r) {
  if (r.index_bytes == 8) write_bounds<long long>(r);
  else write_bounds<int32_t>(r);
}
__global__ __launch_bounds__(64) void expert_bounds_kernel(const Ranges r) { write_ranges(r); }

// WAVES waves a row, four waves a workgroup; a lane takes every 64 WAVES-th multivector, four of them kept from the pass
// that finds the largest entry to the one that writes the codes.  The workgroup behind the rows' writes the bounds of
// `ranges` where there are any (a launch less in front of the products that read them).
template <typename T, int WAVES>
__global__ __launch_bounds__(256) void quantize_rows_kernel(const T* __restrict__ x, int rows, int d,
                                                            unsigned char* __restrict__ codes, float* __restrict__ scale,
                                                            const Ranges ranges) {
  constexpr int RPB = 4 / WAVES, KEEP = 4;
  __shared__ uint32_t s_max[4];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int row = blockIdx.x * RPB + wave / WAVES;
  if (row >= rows) {
    if (ranges.bounds != nullptr && blockIdx.x + 1 == gridDim.x && threadIdx.x < 64) write_ranges(ranges);
    return;
  }
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

// Four waves a row where a row is long, or longer than two loads a lane and rows are few (one wave / four a row, bf16, us: 128
// rows of 128: 2.4 / 2.3, 256: 3.0 / 2.3, 512: 5.2 / 2.6; 2048 rows of 128: 3.4 / 3.7, 256: 5.1 / 4.8, 320: 6.1 / 5.7; 32768
// rows of 128: 23 / 32, 256: 40 / 44, 320: 51 / 52, 512: 85 / 71).  262144 rows of 512 run at 6.1 TB/s (3.2 GB).
// Rows of a launch: a grid holds fewer than 2^32 threads.
constexpr int kLaunchRows = 1 << 22;

template <typename T>
int launch_quantize(const void* x, int rows, int d, void* codes, float* scale, hipStream_t stream, const Ranges& ranges = {}) {
  for (size_t r0 = 0; r0 < (size_t)rows; r0 += kLaunchRows) {
    const int n = (int)std::min<size_t>(rows - r0, kLaunchRows);
    const T* const X = static_cast<const T*>(x) + r0 * d * 8;
    unsigned char* const C = static_cast<unsigned char*>(codes) + r0 * i8_row_bytes(d);
    const Ranges& with = r0 + n == (size_t)rows ? ranges : Ranges{};
    const unsigned more = with.bounds != nullptr, quarter = (unsigned)(n + 3) / 4 + more;
    if (d > 256 || (d > 128 && n <= 2048))
      quantize_rows_kernel<T, 4><<<(unsigned)n + more, 256, 0, stream>>>(X, n, d, C, scale + r0, with);
    else
      quantize_rows_kernel<T, 1><<<quarter, 256, 0, stream>>>(X, n, d, C, scale + r0, with);
    if (check_launch("quantize_rows")) return -1;
  }
  return 0;
}

size_t align256(size_t b) { return (b + 255) & ~(size_t)255; }

// The codes and scales of x's rows, h, the codes and scales of its rows; each on 256 bytes
struct ExpertsAt {
  size_t xq, xs, h, hq, hs, total;
};
ExpertsAt experts_at(size_t x_rows, size_t P, int d, int F) {
  ExpertsAt at;
  at.xq = 0;
  at.xs = at.xq + align256(x_rows * i8_row_bytes(d));
  at.h = at.xs + align256(x_rows * 4);
  at.hq = at.h + align256(P * F * 16);
  at.hs = at.hq + align256(P * i8_row_bytes(F));
  at.total = at.hs + align256(P * 4);
  return at;
}

}  // namespace

size_t int8_experts_bytes(size_t x_rows, size_t P, int d, int F) { return experts_at(x_rows, P, d, F).total; }

namespace {
int run_experts(const void* x, int x_rows, const int32_t* gather, int P, const void* w_up, const float* s_up,
                const float* b_up, const void* w_down, const float* s_down, const float* b_down, const int32_t* offsets,
                int E, int d, int F, int act, void* y, void* workspace, hipStream_t stream, const Ranges& ranges) {
  const ExpertsAt at = experts_at((size_t)x_rows, (size_t)P, d, F);
  char* const b = static_cast<char*>(workspace);
  float *xs = reinterpret_cast<float*>(b + at.xs), *hs = reinterpret_cast<float*>(b + at.hs);
  auto product = [&](const void* q, const float* s, int rows, const int32_t* from, const void* w, const float* sw,
                     const float* bias, int d_in, int d_out, int a, void* to) {
    return (int8_small_pays(P, d_out) ? int8_small_linear : int8_tile_linear)(q, s, rows, from, P, w, sw, bias, offsets, E,
                                                                              d_in, d_out, a, to, kBF16, stream);
  };
  if (launch_quantize<uint16_t>(x, x_rows, d, b + at.xq, xs, stream, ranges)) return -1;
  if (product(b + at.xq, xs, x_rows, gather, w_up, s_up, b_up, d, F, act, b + at.h)) return -1;
  if (launch_quantize<uint16_t>(b + at.h, P, F, b + at.hq, hs, stream)) return -1;
  return product(b + at.hq, hs, P, nullptr, w_down, s_down, b_down, F, d, kActNone, y);
}
}  // namespace

int int8_experts(const void* x, int x_rows, const int32_t* gather, int P, const void* w_up, const float* s_up,
                 const float* b_up, const void* w_down, const float* s_down, const float* b_down, const int32_t* offsets,
                 int E, int d, int F, int act, void* y, void* workspace, hipStream_t stream) {
  return run_experts(x, x_rows, gather, P, w_up, s_up, b_up, w_down, s_down, b_down, offsets, E, d, F, act, y, workspace,
                     stream, Ranges{});
}

size_t int8_rows_bytes(size_t rows, int d) { return rows * i8_row_bytes(d); }

const char* int8_linear_limit(int x_rows, bool gathered, int d_in, int d_out) {
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
  return x_dtype == kF32 ? launch_quantize<float>(x, rows, d, codes, scale, stream)
                         : launch_quantize<uint16_t>(x, rows, d, codes, scale, stream);
}

YGG_API int ygg_int8_grouped_linear(const void* codes, const float* x_scale, int x_rows, const int32_t* gather, int P_max,
                                    const void* w_prepared, const float* w_scale, const float* bias, const int32_t* offsets,
                                    int E, int d_in, int d_out, int act, void* y, int y_dtype, hipStream_t stream) {
  YGG_CHECK_ARG(x_rows >= 0 && P_max >= 0 && E >= 1 && E <= 64 && d_in >= 1 && d_in <= kI8MaxInputs && d_out >= 1,
                "ygg_int8_grouped_linear: bad sizes x_rows=%d P_max=%d E=%d d_in=%d d_out=%d (E <= 64, d_in <= %d)", x_rows,
                P_max, E, d_in, d_out, kI8MaxInputs);
  YGG_CHECK_ARG(act >= kActNone && act <= kActSigmoid, "ygg_int8_grouped_linear: activation %d", act);
  YGG_CHECK_ARG(y_dtype == kF32 || y_dtype == kBF16, "ygg_int8_grouped_linear: output dtype %d unsupported", y_dtype);
  const char* const why = int8_linear_limit(x_rows, gather != nullptr, d_in, d_out);
  YGG_CHECK_ARG(!why, "ygg_int8_grouped_linear: %s (x_rows=%d E=%d d_in=%d d_out=%d)", why, x_rows, E, d_in, d_out);
  if (P_max == 0) return 0;
  YGG_CHECK_ARG(codes && x_scale && w_prepared && w_scale && offsets && y, "ygg_int8_grouped_linear: null pointer");
  YGG_CHECK_ARG(gather || x_rows >= P_max, "ygg_int8_grouped_linear: %d rows of x for %d product rows", x_rows, P_max);
  const size_t yb = (size_t)P_max * d_out * 8 * dtype_size(y_dtype);
  YGG_CHECK_ARG(!overlap(y, yb, codes, int8_rows_bytes((size_t)x_rows, d_in)) && !overlap(y, yb, x_scale, (size_t)x_rows * 4) &&
                    !overlap(y, yb, w_prepared, (size_t)E * i8_expert_bytes(d_out, d_in)) &&
                    !overlap(y, yb, w_scale, (size_t)E * d_out * 4) && !overlap(y, yb, bias, (size_t)E * d_out * 32) &&
                    !overlap(y, yb, gather, (size_t)P_max * 4) && !overlap(y, yb, offsets, (size_t)(E + 1) * 4),
                "ygg_int8_grouped_linear: y must not share memory with an input");
  return (int8_small_pays(P_max, d_out) ? int8_small_linear : int8_tile_linear)(
      codes, x_scale, x_rows, gather, P_max, w_prepared, w_scale, bias, offsets, E, d_in, d_out, act, y, y_dtype, stream);
}

YGG_API int ygg_int8_product_small(int P_max, int d_out) { return int8_small_pays(P_max, d_out); }

YGG_API int ygg_expert_bounds(const void* offsets, const void* counts, int index_bytes, int E, int P, int32_t* bounds,
                              hipStream_t stream) {
  YGG_CHECK_ARG(E >= 1 && E <= 64 && P >= 0, "ygg_expert_bounds: bad sizes E=%d P=%d (E <= 64)", E, P);
  YGG_CHECK_ARG(index_bytes == 4 || index_bytes == 8, "ygg_expert_bounds: indexes of %d bytes", index_bytes);
  YGG_CHECK_ARG(offsets && counts && bounds, "ygg_expert_bounds: null pointer");
  expert_bounds_kernel<<<1, 64, 0, stream>>>(Ranges{offsets, counts, index_bytes, E, P, bounds});
  return check_launch("expert_bounds");
}

YGG_API size_t ygg_int8_grouped_experts_workspace_bytes(int P, int E, int d, int F) {
  return P < 0 || E < 1 || d < 1 || F < 1 ? 0 : int8_experts_bytes((size_t)P, (size_t)P, d, F) + align256((size_t)(E + 1) * 4);
}

YGG_API int ygg_int8_grouped_experts(const void* x_sorted, int P, const void* w_up, const float* s_up, const float* b_up,
                                     const void* w_down, const float* s_down, const float* b_down, const void* offsets,
                                     const void* counts, int index_bytes, int E, int d, int F, int act, void* y,
                                     void* workspace, size_t workspace_bytes, hipStream_t stream) {
  YGG_CHECK_ARG(P >= 0 && E >= 1 && E <= 64 && d >= 1 && F >= 1, "ygg_int8_grouped_experts: bad sizes P=%d E=%d d=%d F=%d (E <= 64)",
                P, E, d, F);
  YGG_CHECK_ARG(act >= kActNone && act <= kActSigmoid, "ygg_int8_grouped_experts: activation %d", act);
  YGG_CHECK_ARG(index_bytes == 4 || index_bytes == 8, "ygg_int8_grouped_experts: indexes of %d bytes", index_bytes);
  const char* why = int8_linear_limit(P, false, d, F);
  if (!why) why = int8_linear_limit(P, false, F, d);
  YGG_CHECK_ARG(!why, "ygg_int8_grouped_experts: %s (P=%d E=%d d=%d F=%d)", why, P, E, d, F);
  if (P == 0) return 0;
  YGG_CHECK_ARG(x_sorted && w_up && s_up && w_down && s_down && offsets && counts && y && workspace,
                "ygg_int8_grouped_experts: null pointer");
  const size_t need = ygg_int8_grouped_experts_workspace_bytes(P, E, d, F), yb = (size_t)P * d * 16;
  YGG_CHECK_ARG(workspace_bytes >= need, "ygg_int8_grouped_experts: workspace of %zu bytes, need %zu", workspace_bytes, need);
  YGG_CHECK_ARG(!overlap(workspace, need, x_sorted, yb) && !overlap(workspace, need, y, yb) &&
                    !overlap(workspace, need, offsets, (size_t)E * index_bytes) &&
                    !overlap(workspace, need, counts, (size_t)E * index_bytes),
                "ygg_int8_grouped_experts: the workspace must not share memory with x_sorted, y or the ranges");
  // (y may be x_sorted, which is read before y is written; nothing else that the products read, nor the workspace)
  const size_t up = (size_t)E * i8_expert_bytes(F, d), down = (size_t)E * i8_expert_bytes(d, F);
  const struct {
    const void* p;
    size_t bytes;
  } kept[] = {{w_up, up},     {s_up, (size_t)E * F * 4},   {b_up, (size_t)E * F * 32},
              {w_down, down}, {s_down, (size_t)E * d * 4}, {b_down, (size_t)E * d * 32}};
  for (const auto& k : kept)
    YGG_CHECK_ARG(!overlap(workspace, need, k.p, k.bytes) && !overlap(y, yb, k.p, k.bytes),
                  "ygg_int8_grouped_experts: y and the workspace must not share memory with the weights, scales or biases");
  int32_t* const bounds =
      reinterpret_cast<int32_t*>(static_cast<char*>(workspace) + int8_experts_bytes((size_t)P, (size_t)P, d, F));
  return run_experts(x_sorted, P, nullptr, P, w_up, s_up, b_up, w_down, s_down, b_down, bounds, E, d, F, act, y, workspace,
                     stream, Ranges{offsets, counts, index_bytes, E, P, bounds});
}
