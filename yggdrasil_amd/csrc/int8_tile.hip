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
// at most N of every wave's memory operations outstanding, every LDS read returned, in all waves
template <int N>
__device__ __forceinline__ void i8_sync() {
  static_assert(N >= 0 && N < 64, "vmcnt field");
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"i"(N) : "memory");
}

template <int YT>
__device__ __forceinline__ void store_blades(const float (&y)[8], __amdgpu_buffer_rsrc_t r, uint32_t off) {
  typedef unsigned int u32x4_t __attribute__((ext_vector_type(4)));
  if constexpr (YT == kBF16) {
    const u32x4_t o = {pack2_bf16(y[0], y[1]), pack2_bf16(y[2], y[3]), pack2_bf16(y[4], y[5]), pack2_bf16(y[6], y[7])};
    __builtin_amdgcn_raw_buffer_store_b128(o, r, off, 0, 0);
  } else {
    u32x4_t lo, hi;
#pragma unroll
    for (int c = 0; c < 4; ++c) lo[c] = __builtin_bit_cast(unsigned, y[c]), hi[c] = __builtin_bit_cast(unsigned, y[4 + c]);
    __builtin_amdgcn_raw_buffer_store_b128(lo, r, off, 0, 0);
    __builtin_amdgcn_raw_buffer_store_b128(hi, r, off + 16, 0, 0);
  }
}

struct I8Tile {
  static constexpr int NT = 256, T = 64, BN = 64;
  static constexpr int A_BYTES = 2 * T * kI8StepBytes;       // 16 KiB: 128 half-rows of a K step
  static constexpr int W_BYTES = BN / 8 * kI8BlockBytes;     // 16 KiB
  static constexpr int STAGE = A_BYTES + W_BYTES;
  // by tile parity: 64 channels' bias and scale, 64 rows' scale and (gathered) place
  static constexpr int BIAS = 0, WS = 2048, XS = WS + 256, IDX = XS + 256, SIDE = IDX + 256;
  static constexpr int SIDE_OFF = 2 * STAGE, LDS = SIDE_OFF + 2 * SIDE;
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
  const __amdgpu_buffer_rsrc_t b_rsrc = rsrc_from(bias, 0, bias ? (uint64_t)E * d_out * 32 : 0);
  const __amdgpu_buffer_rsrc_t ws_rsrc = rsrc_from(ws, 0, (uint64_t)E * d_out * 4);
  uint32_t a_off[4], w_off[4];
  const uint32_t w_lane = (uint32_t)(lane >> 4) * 256 + (2 * (lane & 7) + ((lane >> 3) & 1)) * 16;
  auto side = [&](int n) { return lds0 + C::SIDE_OFF + (n & 1) * C::SIDE; };
  // the rows of tile n that a gather names, asked for before the tile's first loads need them (past the tile's end
  // the last row again)
  auto ask_rows = [&](const Info& t, int n) __attribute__((always_inline)) {
    if (gather && wave == 3)
      i8_dma<4>(rsrc_from(gather, (uint64_t)t.row0 * 4, (uint64_t)(t.row_end - t.row0) * 4), side(n) + C::IDX,
                (uint32_t)min(lane, t.row_end - t.row0 - 1) * 4, 0);
  };
  auto point_at = [&](const Info& t, int n) __attribute__((always_inline)) {
    if (!gather) {  // the tile's rows in place
      const uint64_t first = (uint64_t)t.row0 * half_bytes * 2;
      x_rsrc = rsrc_from(X, first, x_bytes - first);
      s_rsrc = rsrc_from(xs, (uint64_t)t.row0 * 4, (uint64_t)(x_rows - t.row0) * 4);
    }
    w_rsrc = rsrc_from(W, (uint64_t)t.e * expert_bytes, expert_bytes);
    const int* const idx = reinterpret_cast<const int*>(smem + C::SIDE_OFF + (n & 1) * C::SIDE + C::IDX);
    auto source = [&](int tok) { return gather ? idx[tok] : min(tok, t.row_end - t.row0 - 1); };
    // (a place outside x, or behind the last channel, reads zeros)
    if (wave < 2) {
      const int at = wave * 1024 + lane * 16;
      i8_dma<16>(b_rsrc, side(n) + C::BIAS + wave * 1024,
                 t.col0 + (at >> 5) < d_out ? (uint32_t)(t.e * d_out + t.col0) * 32 + at : kBufferOff, 0);
    } else if (wave == 2) {
      i8_dma<4>(ws_rsrc, side(n) + C::WS, t.col0 + lane < d_out ? (uint32_t)(t.e * d_out + t.col0 + lane) * 4 : kBufferOff, 0);
    } else {
      const int own = source(lane);
      i8_dma<4>(s_rsrc, side(n) + C::XS, (unsigned)own < (unsigned)x_rows ? (uint32_t)own * 4 : kBufferOff, 0);
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int q = 4 * wave + u, r = 8 * q + (lane >> 3);
      const int src = source(r >> 1);
      a_off[u] = (unsigned)src < (unsigned)x_rows
                     ? (uint32_t)(2 * src + (r & 1)) * half_bytes + (((lane & 7) ^ (r & 7)) << 4)
                     : kBufferOff;
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

  // The next tile's first step is asked for in the last step of this one, and the rows of the tile after it; the
  // stores of the epilogue come behind them, so the wait for that step leaves them on their way.
  constexpr int kStores = 16 * (YT == kBF16 ? 1 : 2);
  int n = 0, ks = 0, stage = 0;
  Info now = decode(0), next = now;
  ask_rows(now, 0);
  i8_sync<0>();
  point_at(now, 0);
  issue(0, 0);
  if (n_mine > 1) {
    next = decode(1);
    ask_rows(next, 1);
  }
  i8_sync<0>();
  for (;;) {
    const bool last = ks == steps - 1;
    const bool more = n + 1 < n_mine;
    Info after = next;
    if (!last) {
      issue(ks + 1, stage ^ 1);
    } else if (more) {
      point_at(next, n + 1);
      issue(0, stage ^ 1);
      if (n + 2 < n_mine) {
        after = decode(n + 2);
        ask_rows(after, n + 2);
      }
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
      i8_sync<0>();
      continue;
    }
    // the epilogue of tile n: sums to blades in whole numbers, scales and bias, activation
    const int jl = wj * 32 + l32, j = now.col0 + jl;
    const unsigned char* const sd = smem + C::SIDE_OFF + (n & 1) * C::SIDE;
    const float sw = *reinterpret_cast<const float*>(sd + C::WS + jl * 4);
    float bv[8];
#pragma unroll
    for (int c = 0; c < 8; ++c) bv[c] = *reinterpret_cast<const float*>(sd + C::BIAS + jl * 32 + blade_to_mask(c) * 4);
    int vs[2];
#pragma unroll
    for (int a = 0; a < 2; ++a) vs[a] = vsum[a] + __shfl_xor(vsum[a], 32);
    const float* const scale = reinterpret_cast<const float*>(sd + C::XS);
    constexpr int MV_BYTES = YT == kBF16 ? 16 : 32;
    const __amdgpu_buffer_rsrc_t y_rsrc = rsrc_from(Y, (uint64_t)now.row0 * d_out * MV_BYTES,
                                                    (uint64_t)(now.row_end - now.row0) * d_out * MV_BYTES);
#pragma unroll
    for (int rb = 0; rb < 2; ++rb)
#pragma unroll
      for (int q = 0; q < 4; ++q)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int tok = wt * 32 + rb * 16 + 4 * q + 2 * g + h;  // its halves b = 0, 1 are sums v, v + 1
          const int v = 4 * q + 2 * h;
          const auto& s = acc[rb];
          float y[8];
          i8_blades(s[0][0][v] + vs[0], s[0][1][v], s[0][0][v + 1] + vs[0], s[0][1][v + 1], s[1][0][v] + vs[1], s[1][1][v],
                    s[1][0][v + 1] + vs[1], s[1][1][v + 1], sw * scale[tok], bv, y);
          activate_blade<ACT>(y);
          // (a store behind the tile's last row or channel lies past the buffer: every wave stores as often)
          store_blades<YT>(y, y_rsrc, j < d_out ? (uint32_t)(tok * d_out + j) * MV_BYTES : kBufferOff);
        }
    if (!more) break;
    now = next;
    next = after;
    ++n;
    ks = 0;
    i8_sync<kStores>();
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
