// Microscaling (MX) formats: blocks of 32 values along a row that share one power-of-two scale.
//   MX8 rows: e4m3 values; MX4 weights: e2m1 codes (0, .5, 1, 1.5, 2, 3, 4, 6 and their negatives).
//   Scales are e8m0 bytes: byte e stands for 2^(e - 127), 255 for NaN (then the whole block is NaN).
// A block's scale is the smallest power of two with amax <= top * scale (top: 448 of e4m3, 6 of e2m1), so
// that no value saturates; its values are rounded to nearest even.
//
// MX4 weight layout: 16 rows (output features) x 512 columns form one 4352-byte unit, units ordered
// [row tile][column unit]; in a unit, 4 tiles of 128 columns of 1024 bytes each, lane l = (row r = l & 15, g = l >> 4)
// holding 16 bytes at l * 16: the 32 codes of columns 32 g .. 32 g + 31 of the tile (the even one low), one scale
// block; then 64 words, word l byte t the scale of lane l's block of tile t.  So a wave's operand of a 16 x 128 tile
// is one contiguous 1 KiB load, both for the scaled 8-bit matrix instruction (lane (r, g) takes columns 32 g ..)
// and for bf16 ones (step j takes column 32 g + 8 j + i of every g: any order serves that both operands share).
// Rows and columns past the matrix hold zeros.
#pragma once
#include "common.h"

namespace lkv {

constexpr int kMxBlock = 32;
constexpr int kMxUnitCols = 512;
constexpr int kMxTileBytes = 1024;
constexpr int kMxUnitBytes = 4 * kMxTileBytes + 256;

__host__ __device__ inline int64_t mx4_units(int32_t cols) { return (cols + kMxUnitCols - 1) / kMxUnitCols; }

typedef int i32x8 __attribute__((ext_vector_type(8)));

// e8m0 byte of a block with the given |maximum|: exponent minus 8, one more where the mantissa passes 1.75.
__device__ inline int e4m3_scale_byte(double amax) {
  const uint64_t u = __builtin_bit_cast(uint64_t, amax);
  const int ex = static_cast<int>(u >> 52) & 0x7ff;
  if (ex == 0x7ff) return 255;
  const int e = ex - 1023 - 8 + ((u & 0xfffffffffffffull) > 0xc000000000000ull) + 127;
  return e > 254 ? 255 : max(e, 0);
}

__device__ inline double exp2_int(int e) {  // 2^e, -1022 <= e <= 1023
  return __builtin_bit_cast(double, static_cast<uint64_t>(e + 1023) << 52);
}

// fp32 with the last bit odd where the 64-bit value lies between two: a second rounding then rounds the value itself.
__device__ inline float to_odd(double x) {
  const float f = __double2float_rz(x);
  return static_cast<double>(f) == x ? f : __uint_as_float(__float_as_uint(f) | 1u);
}

__device__ inline uint32_t pack_e4m3(float a, float b, float c, float d) {
  const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(c, d, lo, true));
}

// Maximum over the four lanes of a quad (NaN stays).
template <class T>
__device__ inline T quad_max(T x) {
#pragma unroll
  for (int off = 1; off < 4; off <<= 1) {
    const T y = __shfl_xor(x, off);
    x = (x != x || x > y) ? x : y;
  }
  return x;
}

}  // namespace lkv
