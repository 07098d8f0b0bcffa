// int8_tile.hip -- the product of int8 rows with int8 weights (int8_rows.hip: the mathematics and the quantization) for
// enough rows, on v_mfma_i32_32x32x32_i8.
//
// A matrix instruction takes 32 half-rows (16 tokens x column b) against 32 channels of one matrix row a.  Real and
// imaginary parts lie in operands of their own, so the four products of a complex one are
//   Re += U xr,  Re += V ~xi,  Im += U xi,  Im += V xr,
// where ~xi = -xi - 1 (one operation a register; codes stay in int8, -128 to 126): Re is short of sum V, which every
// wave adds up for its channels on the side with four-byte dot products.  A lane ends with all eight reals of its
// multivectors, a channel a lane, so that the epilogue needs no exchange.
//
// Tile: 64 tokens x 64 channels, four waves of 32 x 32 (128 sums a lane), two workgroups a CU, so that one's epilogue
// overlaps the other's products.  K steps of 32 inputs (a line of memory a half-row) go straight to LDS, two stages
// of 32 KiB.  Persistent: a workgroup asks for its next tile's first step before the epilogue of this one.

#include <hip/hip_runtime.h>

#include <algorithm>

#include "int8_rows.h"
#include "pauli_tile.h"
#include "ygg_common.h"

namespace ygg {
namespace {

typedef int i8x16_t __attribute__((ext_vector_type(4)));   // 16 codes
typedef int i32x16_t __attribute__((ext_vector_type(16)));

typedef __attribute__((address_space(3))) void i8_lds_t;
__device__ __forceinline__ uint32_t i8_lds(const unsigned char* p) { return (uint32_t)(uintptr_t)(const i8_lds_t*)p; }
// BYTES (4 or 16) a lane from buffer r at byte off + soff to LDS address lds + BYTES lane.  The off alone decides whether
// a load lies in the buffer; past its end it reads zero.
template <int BYTES>
__device__ __forceinline__ void i8_dma(__amdgpu_buffer_rsrc_t r, uint32_t lds, uint32_t off, uint32_t soff) {
  const uint32_t m0 = __builtin_amdgcn_readfirstlane(lds), so = __builtin_amdgcn_readfirstlane(soff);
  if constexpr (BYTES == 4)
    asm volatile("s_mov_b32 m0, %1\n\tbuffer_load_dword %0, %2, %3 offen lds" ::"v"(off), "s"(m0), "s"(r), "s"(so)
                 : "m0", "memory");
  else
    asm volatile("s_mov_b32 m0, %1\n\tbuffer_load_dwordx4 %0, %2, %3 offen lds" ::"v"(off), "s"(m0), "s"(r), "s"(so)
                 : "m0", "memory");
}
// every direct load landed and every LDS read returned, in all waves
__device__ __forceinline__ void i8_sync() {
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
}

struct I8Tile {
  static constexpr int NT = 256, T = 64, BN = 64;
  static constexpr int A_BYTES = 2 * T * kI8StepBytes;       // 16 KiB: 128 half-rows of a K step
  static constexpr int W_BYTES = BN / 8 * kI8BlockBytes;     // 16 KiB
  static constexpr int STAGE = A_BYTES + W_BYTES;
  static constexpr int S_OFF = 2 * STAGE;                    // 2 x 64 row scales (tile parity)
  static constexpr int LDS = S_OFF + 2 * 256;
};

template <int ACT, int YT>
__global__ __launch_bounds__(I8Tile::NT) __attribute__((amdgpu_waves_per_eu(2))) void int8_tile_kernel(
    const unsigned char* __restrict__ X, uint64_t x_bytes, const float* __restrict__ xs, int x_rows,
    const int32_t* __restrict__ gather, const unsigned char* __restrict__ W, const float* __restrict__ ws,
    const float* __restrict__ bias, const int32_t* __restrict__ offsets, int E, int d_in, int d_out, int P_max,
    void* __restrict__ Y, int n_xcd) {
  using C = I8Tile;
  __shared__ __attribute__((aligned(1024))) unsigned char smem[C::LDS];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wt = wave & 1, wj = wave >> 1;
  const int g = lane >> 5, l32 = lane & 31;

  // lane e: expert e's rows and the tiles before its own
  const int v_beg = min(lane < E ? offsets[lane] : 0, P_max), v_end = min(lane < E ? offsets[lane + 1] : 0, P_max);
  const int v_nt = (v_end - v_beg + C::T - 1) / C::T;
  int v_incl = v_nt;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int v = __shfl_up(v_incl, o);
    if (lane >= o) v_incl += v;
  }
  const int CT = (d_out + C::BN - 1) / C::BN;
  const int n_tiles = __builtin_amdgcn_readlane(v_incl, 63) * CT;
  // one contiguous range of tiles an XCD, a row tile's columns next to each other
  const int per_xcd = gridDim.x / n_xcd;
  const int xcd = blockIdx.x % n_xcd, slot = blockIdx.x / n_xcd;
  const int lo = (int)((long long)n_tiles * xcd / n_xcd), hi = (int)((long long)n_tiles * (xcd + 1) / n_xcd);
  const int n_mine = hi - lo > slot ? (hi - lo - slot + per_xcd - 1) / per_xcd : 0;
  if (n_mine == 0) return;

  const int steps = i8_steps(d_in);
  const uint32_t half_bytes = (uint32_t)steps * kI8StepBytes;   // of a half-row
  const size_t expert_bytes = i8_expert_bytes(d_out, d_in);
  struct Info {
    int e, row0, row_end, col0;
  };
  auto decode = [&](int n) __attribute__((always_inline)) {
    const int L = lo + slot + n * per_xcd;
    const int rt = L / CT;
    const int e = (int)__builtin_ctzll(__ballot(v_incl > rt));
    Info t;
    t.e = e;
    t.row_end = __builtin_amdgcn_readlane(v_end, e);
    t.row0 = __builtin_amdgcn_readlane(v_beg, e) +
             (rt - (__builtin_amdgcn_readlane(v_incl, e) - __builtin_amdgcn_readlane(v_nt, e))) * C::T;
    t.col0 = (L - rt * CT) * C::BN;
    return t;
  };
  auto rsrc_from = [](const void* base, uint64_t off, uint64_t bytes) __attribute__((always_inline)) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(static_cast<const char*>(base)) + off, (short)0,
                                             (uint32_t)(bytes < 0x7fffffffull ? bytes : 0x7fffffffull), kBufferFlags);
  };

  // What the loads of a tile need: this lane's pieces of A (half-rows 8 q + lane / 8 of load q = 4 wave + u, through the
  // swizzle) and of W (load q: 8 channels' U or V, matrix row a in front of the channel).
  const uint32_t lds0 = i8_lds(smem);
  __amdgpu_buffer_rsrc_t x_rsrc = rsrc_from(X, 0, x_bytes), s_rsrc = rsrc_from(xs, 0, (uint64_t)x_rows * 4), w_rsrc = x_rsrc;
  uint32_t a_off[4], w_off[4], s_off = 0;
  const uint32_t w_lane = (uint32_t)(lane >> 4) * 256 + (2 * (lane & 7) + ((lane >> 3) & 1)) * 16;
  auto point_at = [&](const Info& t) __attribute__((always_inline)) {
    if (!gather) {  // the tile's rows in place
      const uint64_t first = (uint64_t)t.row0 * half_bytes * 2;
      x_rsrc = rsrc_from(X, first, x_bytes - first);
      s_rsrc = rsrc_from(xs, (uint64_t)t.row0 * 4, (uint64_t)(x_rows - t.row0) * 4);
    }
    w_rsrc = rsrc_from(W, (uint64_t)t.e * expert_bytes, expert_bytes);
    auto source = [&](int tok) {  // the byte offset of a row of the tile; past its end the last row again
      const int r = min(t.row0 + tok, t.row_end - 1);
      return gather ? gather[r] : r - t.row0;
    };
    const int own = source(lane);
    s_off = !gather || (unsigned)own < (unsigned)x_rows ? (uint32_t)own * 4 : kBufferOff;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int r = 8 * (4 * wave + u) + (lane >> 3);
      const int src = source(r >> 1);
      a_off[u] = !gather || (unsigned)src < (unsigned)x_rows
                     ? (uint32_t)(2 * src + (r & 1)) * half_bytes + (((lane & 7) ^ (r & 7)) << 4)
                     : kBufferOff;
      const int q = 4 * wave + u;
      w_off[u] = (uint32_t)(t.col0 / 8 + (q >> 1)) * steps * kI8BlockBytes + (q & 1) * 1024 + w_lane;
    }
  };
  auto issue = [&](int ks, int stage) __attribute__((always_inline)) {
    const uint32_t at = lds0 + stage * C::STAGE + wave * 4096;
#pragma unroll
    for (int u = 0; u < 4; ++u) i8_dma<16>(x_rsrc, at + u * 1024, a_off[u], (uint32_t)ks * kI8StepBytes);
#pragma unroll
    for (int u = 0; u < 4; ++u) i8_dma<16>(w_rsrc, at + C::A_BYTES + u * 1024, w_off[u], (uint32_t)ks * kI8BlockBytes);
  };

  // this lane's operands in a stage
  const uint32_t a_rd = (uint32_t)(wt * 64 + l32) * 128;
  const uint32_t w_rd = C::A_BYTES + (uint32_t)(wj * 4 + (l32 >> 3)) * kI8BlockBytes + (uint32_t)g * 256 + (l32 & 7) * 16;
  i32x16_t acc[2][2][2];  // [row block][a][re, im]
  int vsum[2];

  int n = 0, ks = 0, stage = 0;
  Info now = decode(0);
  point_at(now);
  issue(0, 0);
  if (wave == 0) i8_dma<4>(s_rsrc, lds0 + C::S_OFF, s_off, 0);
  Info next = now;
  for (;;) {
    i8_sync();
    const bool last = ks == steps - 1;
    const bool more = n + 1 < n_mine;
    if (!last) {
      issue(ks + 1, stage ^ 1);
    } else if (more) {
      next = decode(n + 1);
      point_at(next);
      issue(0, stage ^ 1);
      if (wave == 0) i8_dma<4>(s_rsrc, lds0 + C::S_OFF + ((n + 1) & 1) * 256, s_off, 0);
    }
    if (ks == 0) {
#pragma unroll
      for (int rb = 0; rb < 2; ++rb)
#pragma unroll
        for (int a = 0; a < 2; ++a)
#pragma unroll
          for (int p = 0; p < 2; ++p)
#pragma unroll
            for (int v = 0; v < 16; ++v) acc[rb][a][p][v] = 0;
      vsum[0] = vsum[1] = 0;
    }
    const unsigned char* const st = smem + stage * C::STAGE;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      i8x16_t xr[2], xi[2], xn[2];
#pragma unroll
      for (int rb = 0; rb < 2; ++rb) {
        const unsigned char* p = st + a_rd + rb * 4096;
        xr[rb] = *reinterpret_cast<const i8x16_t*>(p + (((2 * h + g) ^ (l32 & 7)) << 4));
        xi[rb] = *reinterpret_cast<const i8x16_t*>(p + (((4 + 2 * h + g) ^ (l32 & 7)) << 4));
        xn[rb] = ~xi[rb];
      }
#pragma unroll
      for (int a = 0; a < 2; ++a) {
        const i8x16_t u = *reinterpret_cast<const i8x16_t*>(st + w_rd + h * 512 + a * 128);
        const i8x16_t v = *reinterpret_cast<const i8x16_t*>(st + w_rd + 1024 + h * 512 + a * 128);
#pragma unroll
        for (int q = 0; q < 4; ++q) vsum[a] = __builtin_amdgcn_sdot4(v[q], 0x01010101, vsum[a], false);
#pragma unroll
        for (int rb = 0; rb < 2; ++rb) {
          acc[rb][a][0] = __builtin_amdgcn_mfma_i32_32x32x32_i8(xr[rb], u, acc[rb][a][0], 0, 0, 0);
          acc[rb][a][1] = __builtin_amdgcn_mfma_i32_32x32x32_i8(xi[rb], u, acc[rb][a][1], 0, 0, 0);
          acc[rb][a][0] = __builtin_amdgcn_mfma_i32_32x32x32_i8(xn[rb], v, acc[rb][a][0], 0, 0, 0);
          acc[rb][a][1] = __builtin_amdgcn_mfma_i32_32x32x32_i8(xr[rb], v, acc[rb][a][1], 0, 0, 0);
        }
      }
    }
    stage ^= 1;
    if (!last) {
      ++ks;
      continue;
    }
    // the epilogue of tile n: sums to floats, scales, blades, bias, activation
    const int j = now.col0 + wj * 32 + l32;
    constexpr int MV_BYTES = YT == kBF16 ? 16 : 32;
    if (j < d_out) {
      const float sw = ws[(size_t)now.e * d_out + j];
      float bv[8] = {};
      if (bias) {
#pragma unroll
        for (int c = 0; c < 8; ++c) bv[c] = bias[((size_t)now.e * d_out + j) * 8 + blade_to_mask(c)];
      }
      int vs[2];
#pragma unroll
      for (int a = 0; a < 2; ++a) vs[a] = vsum[a] + __shfl_xor(vsum[a], 32);
      const float* const scale = reinterpret_cast<const float*>(smem + C::S_OFF + (n & 1) * 256);
      const uint64_t first = (uint64_t)now.row0 * d_out * MV_BYTES;
      const __amdgpu_buffer_rsrc_t y_rsrc =
          rsrc_from(Y, first, (uint64_t)(now.row_end - now.row0) * d_out * MV_BYTES);
#pragma unroll
      for (int rb = 0; rb < 2; ++rb)
#pragma unroll
        for (int q = 0; q < 4; ++q)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int tok = wt * 32 + rb * 16 + 4 * q + 2 * g + h;  // its halves b = 0, 1 are sums v, v + 1
            if (now.row0 + tok >= now.row_end) continue;
            const int v = 4 * q + 2 * h;
            const float sx = scale[tok];
            auto val = [&](int s) { return i8_value(s, sw, sx); };
            const auto& s = acc[rb];
            pauli_store_mv<ACT, kOutBlade, YT, false>(
                val(s[0][0][v] + vs[0]), val(s[0][1][v]), val(s[0][0][v + 1] + vs[0]), val(s[0][1][v + 1]),
                val(s[1][0][v] + vs[1]), val(s[1][1][v]), val(s[1][0][v + 1] + vs[1]), val(s[1][1][v + 1]), bv, y_rsrc,
                (uint32_t)(tok * d_out + j) * MV_BYTES, 0, d_out, y_rsrc, 0, 0, uint4{});
          }
    }
    if (!more) break;
    now = next;
    ++n;
    ks = 0;
  }
}

template <int ACT, int YT>
int launch_tile(const void* x, const float* xs, int x_rows, const int32_t* gather, int P, const void* w, const float* ws,
                const float* bias, const int32_t* offsets, int E, int d_in, int d_out, void* y, hipStream_t stream) {
  int dev = 0, cus = 256;
  if (hipGetDevice(&dev) != hipSuccess ||
      hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || cus <= 0)
    cus = 256;
  const long long most = ((long long)P / I8Tile::T + std::min(E, P)) * ((d_out + I8Tile::BN - 1) / I8Tile::BN);
  const int xcds = cus % 8 == 0 ? 8 : 1;
  const long long grid = std::min<long long>(2 * cus, (most + xcds - 1) / xcds * xcds);
  int8_tile_kernel<ACT, YT><<<(unsigned)grid, I8Tile::NT, 0, stream>>>(
      static_cast<const unsigned char*>(x), (uint64_t)x_rows * i8_row_bytes(d_in), xs, x_rows, gather,
      static_cast<const unsigned char*>(w), ws, bias, offsets, E, d_in, d_out, P, y, xcds);
  return check_launch("int8_tile");
}

}  // namespace

int int8_tile_linear(const void* x, const float* xs, int x_rows, const int32_t* gather, int P, const void* w, const float* ws,
                     const float* bias, const int32_t* offsets, int E, int d_in, int d_out, int act, void* y, int y_dtype,
                     hipStream_t stream) {
#define YGG_I8(A)                                                                                                          \
  return y_dtype == kF32 ? launch_tile<A, kF32>(x, xs, x_rows, gather, P, w, ws, bias, offsets, E, d_in, d_out, y, stream) \
                         : launch_tile<A, kBF16>(x, xs, x_rows, gather, P, w, ws, bias, offsets, E, d_in, d_out, y, stream)
  switch (act) {
    case kActNone: YGG_I8(kActNone);
    case kActGelu: YGG_I8(kActGelu);
    case kActRelu: YGG_I8(kActRelu);
    default: YGG_I8(kActSigmoid);
  }
#undef YGG_I8
}

}  // namespace ygg
