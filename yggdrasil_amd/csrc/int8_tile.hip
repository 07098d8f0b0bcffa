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
// overlaps the other's products.  A K step is 32 inputs, a line of memory a half-row; its operands go straight to LDS
// (two stages of 32 KiB).  A step's products are four groups, and each group's operands are read from LDS during the
// group before: the first group's during the last of the step before, so the one barrier of a step stands in front of
// its last group, when the step's own operands are all in registers and its stage is free for the step after the next.
// Persistent, one stream of steps over a workgroup's tiles: loads and reads run on through the epilogues.
//
// Bound: with few K steps a tile by the epilogue's vector work (8192 tokens, k = 4, E = 32, 128 -> 512, gelu: 98 us,
// 1.40 POP/s; vector units 56 % of the cycles, matrix units 33 %), with many by the way of the operands through L2
// and LDS (32768 rows, 512 -> 128: 70 us with its codes in the caches, 82 behind the pass that writes them, 1.7 POP/s, 37 %; in
// copies of an earlier step at 81 us, without its loads 62, without its products 78).  No faster, each timed in turn with the kernel
// of its own step (it / that one): rows two steps ahead, up 107 / 103; eight waves of 16 x 32, up 121 / 102, down 81 /
// 74; 64 x 128, one workgroup a CU, three stages, 108 / 102 and 84 / 75.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

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

// A multivector of y to element (row, j) of a tile's rows; a row past the tile's last or a channel j past the last lies
// past the buffer, so every wave stores as often.  fp32 takes two stores: four lanes exchange theirs so that each is 64
// bytes a quad instead of every second 16.
template <int YT, bool STREAM>
__device__ __forceinline__ void store_blades(const float (&y)[8], __amdgpu_buffer_rsrc_t r, int row, int j, int d_out) {
  typedef unsigned int u32x4_t __attribute__((ext_vector_type(4)));
  constexpr int kPolicy = STREAM ? 2 : 0;
  if constexpr (YT == kBF16) {
    const u32x4_t o = {pack2_bf16(y[0], y[1]), pack2_bf16(y[2], y[3]), pack2_bf16(y[4], y[5]), pack2_bf16(y[6], y[7])};
    __builtin_amdgcn_raw_buffer_store_b128(o, r, j < d_out ? (uint32_t)(row * d_out + j) * 16 : kBufferOff, 0, kPolicy);
  } else {
    constexpr int kLow = 0x50, kHigh = 0xFA;  // lanes 0 0 1 1 and 2 2 3 3 of a quad
    const bool odd = threadIdx.x & 1;
    u32x4_t first, second;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const int lo = __builtin_bit_cast(int, y[c]), hi = __builtin_bit_cast(int, y[4 + c]);
      const int f0 = __builtin_amdgcn_mov_dpp(lo, kLow, 0xf, 0xf, true), f1 = __builtin_amdgcn_mov_dpp(hi, kLow, 0xf, 0xf, true);
      const int s0 = __builtin_amdgcn_mov_dpp(lo, kHigh, 0xf, 0xf, true), s1 = __builtin_amdgcn_mov_dpp(hi, kHigh, 0xf, 0xf, true);
      first[c] = (unsigned)(odd ? f1 : f0);
      second[c] = (unsigned)(odd ? s1 : s0);
    }
    const int j0 = (j & ~3) + ((j >> 1) & 1);  // the multivectors that this lane stores a half of: j0 and j0 + 2
    const uint32_t at = (uint32_t)(row * d_out + j0) * 32 + (odd ? 16 : 0);
    __builtin_amdgcn_raw_buffer_store_b128(first, r, j0 < d_out ? at : kBufferOff, 0, kPolicy);
    __builtin_amdgcn_raw_buffer_store_b128(second, r, j0 + 2 < d_out ? at + 64 : kBufferOff, 0, kPolicy);
  }
}

struct I8Tile {
  static constexpr int NT = 256, T = 64, BN = 64;
  static constexpr int A_BYTES = 2 * T * kI8StepBytes;    // 16 KiB: 128 half-rows of a K step
  static constexpr int W_BYTES = BN / 8 * kI8BlockBytes;  // 16 KiB
  static constexpr int STAGE = A_BYTES + W_BYTES;
  // three tiles' bias and scale of 64 channels and scale of 64 rows, two tiles' (gathered) places of 64 rows
  static constexpr int BIAS = 0, WS = 2048, XS = WS + 256, SIDE = XS + 256;
  static constexpr int SIDE_OFF = 2 * STAGE, IDX_OFF = SIDE_OFF + 3 * SIDE, LDS = IDX_OFF + 2 * 256;
  static_assert(LDS <= 80 * 1024, "two workgroups a CU");
};

// A tile.  The sums of block `which` (tokens 16 which .. of a wave's 32) alone where `half`; `compact`: an expert's last
// rows, at most 32, laid into the tokens of block 0.
struct I8Item {
  int e, row0, row_end, col0;
  bool half, compact;
  int which;
};

template <int ACT, int YT, bool STREAM>
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

  // lane e: expert e's rows, and the tiles up to its last: whole ones, and short last ones ("compact", half the products)
  auto inside = [&](int at) { return lane < E ? min(max(offsets[lane + at], 0), P_max) : 0; };
  const int v_beg = inside(0), v_end = max(inside(1), v_beg);
  const int v_all = (v_end - v_beg + C::T - 1) / C::T;
  const int v_short = v_all > 0 && v_end - v_beg - (v_all - 1) * C::T <= C::T / 2 ? 1 : 0;
  const int v_nt = v_all - v_short;
  int v_incl = v_nt, v_sincl = v_short;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int p = __shfl_up(v_incl, o), q = __shfl_up(v_sincl, o);
    if (lane >= o) v_incl += p, v_sincl += q;
  }
  // One contiguous range of each list an XCD, a row tile's columns next to each other: the whole tiles in rounds over
  // the XCD's workgroups, then items of half the work -- the compact tiles, and the whole tiles of the last round cut
  // in halves where these still fit in one --, from the first workgroup that has a whole tile less.
  const int CT = (d_out + C::BN - 1) / C::BN;
  const int n_whole = __builtin_amdgcn_readlane(v_incl, 63) * CT, n_short = __builtin_amdgcn_readlane(v_sincl, 63) * CT;
  const int per_xcd = gridDim.x / n_xcd;
  const int xcd = blockIdx.x % n_xcd, slot = blockIdx.x / n_xcd;
  auto cut = [&](int n, int x) { return (int)((long long)n * x / n_xcd); };
  const int lo = cut(n_whole, xcd), R = cut(n_whole, xcd + 1) - lo;
  const int slo = cut(n_short, xcd), n_shorts = cut(n_short, xcd + 1) - slo;
  const int rounds = R / per_xcd, rem = R - rounds * per_xcd;
  const bool split = rem > 0 && 2 * rem <= per_xcd;
  const int n_full = rounds + (!split && slot < rem ? 1 : 0);
  const int n_items = n_shorts + (split ? 2 * rem : 0);
  const int rank = split || slot >= rem ? slot - (split ? 0 : rem) : slot - rem + per_xcd;
  const int n_mine = n_full + (n_items > rank ? (n_items - rank + per_xcd - 1) / per_xcd : 0);
  if (n_mine == 0) return;

  auto decode = [&](int n) __attribute__((always_inline)) {
    const int item = n - n_full < 0 ? -1 : rank + (n - n_full) * per_xcd;
    I8Item t;
    t.half = item >= 0;
    t.compact = item >= 0 && item < n_shorts;
    const int L = t.compact ? slo + item : item >= 0 ? lo + rounds * per_xcd + ((item - n_shorts) >> 1) : lo + slot + n * per_xcd;
    t.which = t.half && !t.compact ? (item - n_shorts) & 1 : 0;
    const int rt = L / CT;
    t.col0 = (L - rt * CT) * C::BN;
    t.e = (int)__builtin_ctzll(__ballot((t.compact ? v_sincl : v_incl) > rt));
    const int beg = __builtin_amdgcn_readlane(v_beg, t.e);
    const int whole = __builtin_amdgcn_readlane(v_nt, t.e);
    t.row_end = __builtin_amdgcn_readlane(v_end, t.e);
    t.row0 = beg + (t.compact ? whole : rt - (__builtin_amdgcn_readlane(v_incl, t.e) - whole)) * C::T;
    return t;
  };
  auto rsrc_from = [](const void* base, uint64_t off, uint64_t bytes) __attribute__((always_inline)) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(static_cast<const char*>(base)) + off, (short)0,
                                             (uint32_t)(bytes < 0x7fffffffull ? bytes : 0x7fffffffull), kBufferFlags);
  };

  const int steps = i8_steps(d_in);
  const uint32_t half_bytes = (uint32_t)steps * kI8StepBytes;  // of a half-row
  const size_t expert_bytes = i8_expert_bytes(d_out, d_in);
  const uint32_t lds0 = i8_lds(smem);
  __amdgpu_buffer_rsrc_t x_rsrc = rsrc_from(X, 0, x_bytes), s_rsrc = rsrc_from(xs, 0, (uint64_t)x_rows * 4), w_rsrc = x_rsrc;
  const __amdgpu_buffer_rsrc_t b_rsrc = rsrc_from(bias, 0, bias ? (uint64_t)E * d_out * 32 : 0);
  const __amdgpu_buffer_rsrc_t ws_rsrc = rsrc_from(ws, 0, (uint64_t)E * d_out * 4);

  // The rows that a gather names, asked for a tile before the tile's own loads need them (past the tile's end the last
  // row again).  Token slot t of a tile is its row t, or of a compact one row 16 (t / 32) + t % 16.
  auto ask_rows = [&](const I8Item& t, int n) __attribute__((always_inline)) {
    if (gather && wave == 3) {
      const int row = t.compact ? (lane >> 5) * 16 + (lane & 15) : lane;
      i8_dma<4>(rsrc_from(gather, (uint64_t)t.row0 * 4, (uint64_t)(t.row_end - t.row0) * 4), lds0 + C::IDX_OFF + (n & 1) * 256,
                (uint32_t)min(row, t.row_end - t.row0 - 1) * 4, 0);
    }
  };
  // What the row loads of a tile need -- this lane's pieces are half-rows 8 q + lane / 8 of load q = 4 wave + u, through
  // the swizzle --, and the loads of its side.  A place outside x, behind the last channel or in a block that is not
  // computed reads zeros, without traffic.
  uint32_t a_off[4];
  auto point_rows = [&](const I8Item& t, int n) __attribute__((always_inline)) {
    if (!gather) {  // the tile's rows in place
      const uint64_t first = (uint64_t)t.row0 * half_bytes * 2;
      x_rsrc = rsrc_from(X, first, x_bytes - first);
      s_rsrc = rsrc_from(xs, (uint64_t)t.row0 * 4, (uint64_t)(x_rows - t.row0) * 4);
    }
    const int* const idx = reinterpret_cast<const int*>(smem + C::IDX_OFF + (n & 1) * 256);
    auto source = [&](int tok) {
      const int row = t.compact ? (tok >> 5) * 16 + (tok & 15) : tok;
      const int src = gather ? idx[tok] : min(row, t.row_end - t.row0 - 1);
      return t.half && ((tok >> 4) & 1) != t.which ? -1 : src;
    };
    const uint32_t side = lds0 + C::SIDE_OFF + (n % 3) * C::SIDE;
    if (wave < 2) {
      const int at = wave * 1024 + lane * 16;
      i8_dma<16>(b_rsrc, side + C::BIAS + wave * 1024,
                 t.col0 + (at >> 5) < d_out ? (uint32_t)(t.e * d_out + t.col0) * 32 + at : kBufferOff, 0);
    } else if (wave == 2) {
      i8_dma<4>(ws_rsrc, side + C::WS, t.col0 + lane < d_out ? (uint32_t)(t.e * d_out + t.col0 + lane) * 4 : kBufferOff, 0);
    } else {
      const int own = source(lane);
      i8_dma<4>(s_rsrc, side + C::XS, (unsigned)own < (unsigned)x_rows ? (uint32_t)own * 4 : kBufferOff, 0);
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int r = 8 * (4 * wave + u) + (lane >> 3);
      const int src = source(r >> 1);
      a_off[u] = (unsigned)src < (unsigned)x_rows
                     ? (uint32_t)(2 * src + (r & 1)) * half_bytes + (((lane & 7) ^ ((r >> 1) & 7)) << 4)
                     : kBufferOff;
    }
  };
  // Weights: load q = 4 wave + u of a K step is 8 channels' U or V, 16 bytes of matrix row a and channel jj from (g, n =
  // 2 jj + a); an odd block of channels has its rows a exchanged, so that 16 lanes of a read meet all banks.
  uint32_t w_off[4];
  auto point_weights = [&](const I8Item& t) __attribute__((always_inline)) {
    w_rsrc = rsrc_from(W, (uint64_t)t.e * expert_bytes, expert_bytes);
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int q = 4 * wave + u, a = ((lane >> 3) ^ (q >> 1)) & 1;
      w_off[u] = (uint32_t)(t.col0 / 8 + (q >> 1)) * steps * kI8BlockBytes + (q & 1) * 1024 + (lane >> 4) * 256 +
                 (2 * (lane & 7) + a) * 16;
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
  uint32_t a_rd[2], w_rd[2];  // [h] (the imaginary parts at ^ 64), [a]
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    a_rd[h] = (uint32_t)(wt * 64 + l32) * 128 + (((2 * h + g) ^ ((l32 >> 1) & 7)) << 4);
    w_rd[h] = C::A_BYTES + (uint32_t)(wj * 4 + (l32 >> 3)) * kI8BlockBytes + (uint32_t)g * 256 + ((h ^ (l32 >> 3)) & 1) * 128 +
              (l32 & 7) * 16;
  }
  i32x16_t acc[2][2][2];  // [row block][a][re, im]
  int vsum[2];
  // A K step's products: group (h, a) is 16 inputs, one matrix row of the weights.  Where `half`, one row block.
  i8x16_t xr[2][2], xi[2][2], u[2], v[2];  // [h][rb], [a]
  auto read = [&](uint32_t at, const I8Item& t, int grp) __attribute__((always_inline)) {
    const int h = grp >> 1, a = grp & 1;
    const unsigned char* const st = smem + at;
    if (a == 0) {
      const uint32_t block = t.half ? t.which * 4096 : 0;
#pragma unroll
      for (int rb = 0; rb < 2; ++rb) {
        xr[h][rb] = *reinterpret_cast<const i8x16_t*>(st + block + a_rd[h] + rb * 4096);
        xi[h][rb] = *reinterpret_cast<const i8x16_t*>(st + block + (a_rd[h] ^ 64) + rb * 4096);
      }
    }
    u[a] = *reinterpret_cast<const i8x16_t*>(st + w_rd[a] + h * 512);
    v[a] = *reinterpret_cast<const i8x16_t*>(st + w_rd[a] + h * 512 + 1024);
  };
  auto multiply = [&](bool half, int grp, auto first_tag) __attribute__((always_inline)) {
    const int h = grp >> 1, a = grp & 1;
    const bool zero = decltype(first_tag)::value && h == 0;
    auto block = [&](int rb) __attribute__((always_inline)) {
      acc[rb][a][0] = __builtin_amdgcn_mfma_i32_32x32x32_i8(xr[h][rb], u[a], zero ? i32x16_t{} : acc[rb][a][0], 0, 0, 0);
      acc[rb][a][1] = __builtin_amdgcn_mfma_i32_32x32x32_i8(xi[h][rb], u[a], zero ? i32x16_t{} : acc[rb][a][1], 0, 0, 0);
      acc[rb][a][0] = __builtin_amdgcn_mfma_i32_32x32x32_i8(~xi[h][rb], v[a], acc[rb][a][0], 0, 0, 0);
      acc[rb][a][1] = __builtin_amdgcn_mfma_i32_32x32x32_i8(xr[h][rb], v[a], acc[rb][a][1], 0, 0, 0);
    };
    block(0);
    if (zero) vsum[a] = 0;
#pragma unroll
    for (int q = 0; q < 4; ++q) vsum[a] = __builtin_amdgcn_sdot4(v[a][q], 0x01010101, vsum[a], false);
    if (!half) block(1);
    __builtin_amdgcn_sched_barrier(0);
  };

  // The stream of K steps: c is the next step to be asked for, two ahead of the products.
  I8Item ct = decode(0);
  int cn = 0, cks = 0;
  auto ask = [&](int stage) __attribute__((always_inline)) {
    if (cn >= n_mine) return;
    if (cks == 0) {
      point_rows(ct, cn);
      point_weights(ct);
    }
    issue(cks, stage);
    if (++cks == steps) {
      cks = 0;
      if (++cn < n_mine) {
        ct = decode(cn);
        ask_rows(ct, cn);
      }
    }
  };
  ask_rows(ct, 0);
  i8_sync<0>();
  ask(0);
  i8_sync<0>();
  ask(1);
  // At a step's barrier the loads of the step after it have landed: behind them come only the stores of an epilogue in
  // between, which stay on their way.
  constexpr int kStores = 16 * (YT == kBF16 ? 1 : 2);
  I8Item t = decode(0), next = t;
  read(0, t, 0);
  int stage = 0;
  bool stores = false;
  for (int n = 0;; ++n) {
    const bool more = n + 1 < n_mine;
    if (more) next = decode(n + 1);
    auto k_step = [&](bool last, auto first_tag) __attribute__((always_inline)) {
      const uint32_t at = stage * C::STAGE;
      __builtin_amdgcn_s_setprio(2);
#pragma unroll
      for (int grp = 0; grp < 3; ++grp) {
        read(at, t, grp + 1);
        multiply(t.half, grp, first_tag);
      }
      if (!last || more) {
        if (stores) i8_sync<kStores>();
        else i8_sync<0>();
        stores = false;
        ask(stage);
        stage ^= 1;
        read(stage * C::STAGE, last ? next : t, 0);
      }
      multiply(t.half, 3, first_tag);
      __builtin_amdgcn_s_setprio(0);
    };
    k_step(steps == 1, std::true_type{});
#pragma unroll 1
    for (int ks = 1; ks < steps; ++ks) k_step(ks == steps - 1, std::false_type{});
    {
      // the epilogue: sums to blades in whole numbers, scales and bias, activation
      const int jl = wj * 32 + l32, j = t.col0 + jl;
      const unsigned char* const sd = smem + C::SIDE_OFF + (n % 3) * C::SIDE;
      const float sw = *reinterpret_cast<const float*>(sd + C::WS + jl * 4);
      float bv[8];
#pragma unroll
      for (int c = 0; c < 8; ++c) bv[c] = *reinterpret_cast<const float*>(sd + C::BIAS + jl * 32 + blade_to_mask(c) * 4);
      int vs[2];
#pragma unroll
      for (int a = 0; a < 2; ++a) vs[a] = vsum[a] + __shfl_xor(vsum[a], 32);
      constexpr int MV_BYTES = YT == kBF16 ? 16 : 32;
      const __amdgpu_buffer_rsrc_t y_rsrc = rsrc_from(Y, (uint64_t)t.row0 * d_out * MV_BYTES,
                                                      (uint64_t)(t.row_end - t.row0) * d_out * MV_BYTES);
#pragma unroll
      for (int rb = 0; rb < 2; ++rb) {
        if (rb == 1 && t.half) break;
        const int tok0 = wt * 32 + (t.half ? t.which : rb) * 16;             // token slot of the block's first row
        const int row0 = (t.compact ? wt * 16 : tok0) + 2 * g;               // its row in the tile, this lane's first
        const float* const scale = reinterpret_cast<const float*>(sd + C::XS) + tok0 + 2 * g;
#pragma unroll
        for (int q = 0; q < 4; ++q)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int v = 4 * q + 2 * h;  // the halves b = 0, 1 of row 4 q + h are sums v, v + 1
            const auto& s = acc[rb];
            float y[8];
            i8_blades(s[0][0][v] + vs[0], s[0][1][v], s[0][0][v + 1] + vs[0], s[0][1][v + 1], s[1][0][v] + vs[1], s[1][1][v],
                      s[1][0][v + 1] + vs[1], s[1][1][v + 1], sw * scale[4 * q + h], bv, y);
            activate_blade<ACT>(y);
            store_blades<YT, STREAM>(y, y_rsrc, row0 + 4 * q + h, j, d_out);
          }
      }
    }
    if (!more) break;
    stores = !t.half;  // (a half tile's are fewer: the next wait takes them in)
    t = next;
  }
}

template <int ACT, int YT>
int launch_tile(const void* x, const float* xs, int x_rows, const int32_t* gather, int P, const void* w, const float* ws,
                const float* bias, const int32_t* offsets, int E, int d_in, int d_out, void* y, hipStream_t stream) {
  int dev = 0, cus = 256;
  if (hipGetDevice(&dev) != hipSuccess ||
      hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || cus <= 0)
    cus = 256;
  // never more workgroups than items can exist (a tile may be cut in two)
  const long long tiles = ((long long)P / I8Tile::T + std::min(E, P)) * ((d_out + I8Tile::BN - 1) / I8Tile::BN);
  const int xcds = cus % 8 == 0 ? 8 : 1;
  const long long grid = std::min<long long>(2 * cus, (2 * tiles + xcds - 1) / xcds * xcds);
  // bf16 outputs go past L2: their stores are whole lines (a product with L2's usual policy / so, us: 2048 rows, 128 ->
  // 512: 13.7 / 12.6, 32768, E = 32: 111 / 88; 512 -> 128 70.5 / 69.7, with the combine that reads its rows next 86.6 / 88;
  // layers of 2048 tokens, 128-512, E = 32, k = 2 73.0 / 69.4, 8192, k = 4 298 / 289.5, 4096, 256-1024, E = 64, k = 2
  // 255 / 253.5, 512-2048, E = 16 677 / 674.7).  fp32 ones do where they are far more than the caches behind it hold (128 ->
  // 512: 67 MB 21.6 / 24.8, 134 MB 40 / 46, 268 MB 81 / 75, 537 MB 170 / 144).
  const bool stream_out = YT == kBF16 || (uint64_t)P * d_out * 32 > (uint64_t)192 << 20;
  auto* const kernel = stream_out ? int8_tile_kernel<ACT, YT, true> : int8_tile_kernel<ACT, YT, YT == kBF16>;
  kernel<<<(unsigned)grid, I8Tile::NT, 0, stream>>>(
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
