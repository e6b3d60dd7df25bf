// Microscaling (MX) formats: blocks of 32 values along a row that share one power-of-two scale.
//   MX8 rows: e4m3 values; MX4 weights: e2m1 codes (0, .5, 1, 1.5, 2, 3, 4, 6 and their negatives).
//   Scales are e8m0 bytes: byte e stands for 2^(e - 127), 255 for NaN (then the whole block is NaN).
// A block's scale is the smallest power of two with amax <= top * scale (top: 448 of e4m3, 6 of e2m1), so
// that no value saturates; its values are rounded to nearest even.
#pragma once
#include "common.h"
#include "mx_layout.h"

namespace lkv {

constexpr int kMxBlock = 32;

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

template <int kCtrl>
__device__ inline float quad_swap(float x) {
  return __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(x), kCtrl, 0xf, 0xf, true));
}

// Maximum over the four lanes of a quad (NaN stays).
__device__ inline float quad_max(float x) {
  x = fmax_nan(x, quad_swap<0xb1>(x));  // lanes 1 0 3 2
  return fmax_nan(x, quad_swap<0x4e>(x));  // lanes 2 3 0 1
}

__device__ inline double quad_max(double x) {
#pragma unroll
  for (int off = 1; off < 4; off <<= 1) {
    const double y = __shfl_xor(x, off);
    x = (x != x || x > y) ? x : y;
  }
  return x;
}

// Eight values of a lane whose quad holds one block as e4m3 bytes, and the block's scale byte: correctly rounded values of
// the real ones, which y holds within a relative kMxError.  Almost always that decides: the scale where |maximum| is not
// that near 1.75 times a power of two, the bytes where both ends of a value's interval round alike.  Elsewhere (2e-5 of
// the values, and what leaves fp32's range or is NaN) exact(d) gives the eight in 64 bits, whose own error reaches
// another border once in 10^12.  A lane makes its quad take that path with y[0] = NaN.
constexpr float kMxError = 0x1p-20f;
template <class F>
__device__ inline uint2 quantize_e4m3(const float (&y)[8], int& byte, F&& exact) {
  float m = fmax_nan(fabsf(y[0]), fabsf(y[1]));
#pragma unroll
  for (int j = 2; j < 8; j += 2) m = fmax3_nan(m, fabsf(y[j]), fabsf(y[j + 1]));
  const uint32_t bits = __float_as_uint(quad_max(m));
  const int ex = static_cast<int>(bits >> 23);  // (the sign is clear)
  const bool wide = ex < 30 || ex > 250 || ((bits - 0x600000u + 16u) & 0x7fffffu) <= 32u;
  byte = ex - 8 + ((bits & 0x7fffffu) > 0x600000u);
  const float f = __uint_as_float(static_cast<uint32_t>(254 - byte) << 23);
  const float lo = f * (1.f - kMxError), hi = f * (1.f + kMxError);
  uint2 q = make_uint2(pack_e4m3(y[0] * lo, y[1] * lo, y[2] * lo, y[3] * lo),
                       pack_e4m3(y[4] * lo, y[5] * lo, y[6] * lo, y[7] * lo));
  const uint2 p = make_uint2(pack_e4m3(y[0] * hi, y[1] * hi, y[2] * hi, y[3] * hi),
                             pack_e4m3(y[4] * hi, y[5] * hi, y[6] * hi, y[7] * hi));
  if (wide || q.x != p.x || q.y != p.y) {
    double d[8];
    exact(d);
    if (wide) {  // (the same for the quad)
      double a = fabs(d[0]);
#pragma unroll
      for (int j = 1; j < 8; ++j) a = (a != a || a > fabs(d[j])) ? a : fabs(d[j]);
      byte = e4m3_scale_byte(quad_max(a));
    }
    if (byte == 255) return make_uint2(0, 0);
    const double g = exp2_int(127 - byte);
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = to_odd(d[j] * g);
    q = make_uint2(pack_e4m3(v[0], v[1], v[2], v[3]), pack_e4m3(v[4], v[5], v[6], v[7]));
  }
  return q;
}

}  // namespace lkv
