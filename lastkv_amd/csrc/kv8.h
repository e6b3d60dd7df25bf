// The shared cache in 8 bits: 32-token blocks of e4m3 codes, 4096 bytes a (page, kv head), K and V apart, each block with one
// scale byte e that stands for 2^(e - 127) (255: the block is NaN).  The value of code c is c * 2^(e - 127), exact in bf16.
//
// Layout of a block: 4 pieces of 64 lanes x 16 bytes, so that a wave reads 1 KiB with each load and every lane gets the
// matrix operands that the bf16 layout gives it (common.h), two of them a load:
//   K element (w, d): piece u * 2 + (d >> 6), lane ((d >> 3) & 3) * 16 + r, byte ((d >> 5) & 1) * 8 + (d & 7)
//     with u = (w >> 2) & 1, r = ((w >> 3) << 2) | (w & 3): bf16 operands kb = 2 (d >> 6) and the next.
//   V element (w, d): piece d >> 5, lane (w >> 3) * 16 + (d & 15), byte ((d >> 4) & 1) * 8 + (w & 7):
//     bf16 operands nb = 2 (d >> 5) and the next.
#pragma once
#include "common.h"
#include "runtime.h"

namespace lkv {

constexpr int kKv8Block = kBlockElems;  // bytes of a block

// An 8-bit page pool on the device.
struct Kv8Pool {
  const uint8_t* k;
  const uint8_t* v;
  const uint8_t* ks;  // scale of (page p, head h): ks[h * s_hs + p]
  const uint8_t* vs;
  int64_t page, hs, s_hs;  // bytes
  int32_t pages;
};

// Checks an lkv_kv8_pool (no device calls) and copies it.
int32_t kv8_pool(const lkv_kv8_pool* a, const char* name, Kv8Pool& p);

__device__ inline float kv8_scale(uint32_t byte) {  // (0 and 255 set the mantissa's top bit: 2^-127 and NaN)
  return __uint_as_float(byte << 23 | (((byte + 1) & 0xfeu) == 0 ? 0x400000u : 0u));
}

// The first n of eight bf16 values, the others 0.
__device__ inline uint4 keep_tokens(uint4 x, int n) {
  const auto mask = [n](int i) { return n >= 2 * i + 2 ? 0xffffffffu : n == 2 * i + 1 ? 0xffffu : 0u; };
  return make_uint4(x.x & mask(0), x.y & mask(1), x.z & mask(2), x.w & mask(3));
}

// Eight e4m3 codes times a power of two as eight bf16 values.
__device__ inline uint4 kv8_to_bf16(uint32_t lo, uint32_t hi, float scale) {
  return make_uint4(__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, false)),
                    __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, true)),
                    __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, false)),
                    __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, true)));
}

}  // namespace lkv
