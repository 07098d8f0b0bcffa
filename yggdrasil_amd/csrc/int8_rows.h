// int8_rows.h -- the layout of quantized rows and of the int8 Pauli weights that they meet.
#pragma once

#include "pauli_common.h"

namespace ygg {

// A multivector's halved Pauli matrix holds 8 reals: entries (c, b), real and imaginary parts.  A quantized row keeps them
// as int8 codes with one scale a row (both columns b): for b = 0, 1 and every 32 inputs (a K step), 128 bytes
//   [re, im][g 4][16 bytes]: byte 2 m + c holds the code of entry (c, b) of input 32 ks + 8 g + m,
// zero past the row's last input.  One 16-byte run is a lane's operand of v_mfma_i32_32x32x32_i8 -- real and imaginary
// parts lie in runs of their own, so the rotation by i exchanges two registers instead of bytes -- and a K step
// of a half-row is one line of memory.
constexpr int kI8Step = 32;         // inputs of a K step
constexpr int kI8StepBytes = 128;   // a half-row's bytes of it
__host__ __device__ inline int i8_steps(int d) { return (d + kI8Step - 1) / kI8Step; }
__host__ __device__ inline size_t i8_row_bytes(int d) { return (size_t)i8_steps(d) * 2 * kI8StepBytes; }

// The weights of format 5 (decode_pauli.hip): per expert [ceil(d_out / 8)][K steps][U, V][g 4][n 16][16 bytes],
// n = 2 jj + a (channel 8 jb + jj, matrix row a), byte 2 m + c the code of entry (a, c), the inputs as above.
constexpr int kI8BlockBytes = 2048;  // 8 channels of a K step
__host__ __device__ inline size_t i8_expert_bytes(int d_out, int d_in) {
  return (size_t)((d_out + 7) / 8) * i8_steps(d_in) * kI8BlockBytes;
}
// The blades of an output multivector from the sums of its halved matrix (entry a b, re and im): sums and differences of
// two of them, still whole numbers, then one rounding to fp32, the two scales' product and the bias in one multiply-add.
// The same in every kernel, so a row's outputs do not depend on which takes its batch.  (A product of scales below
// 2^-126, which takes rows or weights near their own lower limits, loses bits; one past fp32's largest is infinite.)
__device__ __forceinline__ void i8_blades(int r00, int i00, int r01, int i01, int r10, int i10, int r11, int i11, float scale,
                                          const float (&bias)[8], float (&y)[8]) {
  const int t[8] = {r00 + r11, r10 + r01, i10 - i01, r00 - r11, i00 - i11, r10 - r01, i10 + i01, i00 + i11};
#pragma unroll
  for (int c = 0; c < 8; ++c) y[c] = __builtin_fmaf((float)t[c], scale, bias[c]);
}

// Sums and differences of two sums of 4 d_in products of codes (up to 127, and -128 where a code is complemented) stay
// below 2^31
constexpr int kI8MaxInputs = 16384;

}  // namespace ygg
