// Projections over MX4 weights (layout in mx.h): y[m][n] = bf16(sum_k x[m][k] w[n][k] + bias[n]), x in bf16 or MX8
// rows, and the layout's packing.
#include <algorithm>

#include "mx.h"
#include "runtime.h"

namespace lkv {
namespace {

struct LinearParams {
  const uint8_t* w;
  const void* x;
  int64_t x_stride;  // elements
  const uint8_t* xs;
  int64_t xs_stride;
  const uint16_t* bias;
  uint16_t* out;
  int64_t out_stride;
  int32_t M, N, K;
  int32_t units;
};

constexpr int kWaves = 8;

__device__ inline float e8m0(uint32_t word, int t) {  // the scale's exponent in place (0: read as 2^-127 by the convert)
  return __uint_as_float(((word >> (8 * t)) & 0xffu) << 23);
}

// Eight codes of a word as scaled bf16 (exact: 2 significant bits, bf16's exponents).
__device__ inline uint4 e2m1_to_bf16(uint32_t codes, float scale) {
  return make_uint4(__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 0)),
                    __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 1)),
                    __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 2)),
                    __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 3)));
}

// One workgroup per (NT row tiles of the weight, MT tiles of 16 rows of x); its 8 waves take every eighth unit of 512
// columns and their sums are added through LDS, in the waves' order.
template <bool kMx8, int MT, int NT>
__global__ __launch_bounds__(kWaves * 64) void mx4_rows_kernel(const LinearParams p) {
  __shared__ f32x4 part[kWaves][MT][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int r = lane & 15, g = lane >> 4;
  const int nt0 = blockIdx.x * NT, m0 = blockIdx.y * (16 * MT);
  const int ntiles = (p.N + 15) >> 4;
  f32x4 acc[NT][MT];
#pragma unroll
  for (int i = 0; i < NT; ++i)
#pragma unroll
    for (int j = 0; j < MT; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  int64_t row[MT];
#pragma unroll
  for (int j = 0; j < MT; ++j) row[j] = min(m0 + 16 * j + r, p.M - 1);  // (rows past the last repeat it and are not stored)
  const uint8_t* w[NT];
#pragma unroll
  for (int i = 0; i < NT; ++i) w[i] = p.w + static_cast<int64_t>(min(nt0 + i, ntiles - 1)) * p.units * kMxUnitBytes;
  for (int u = wave; u < p.units; u += kWaves) {
    uint32_t ws[NT];
#pragma unroll
    for (int i = 0; i < NT; ++i)
      ws[i] = *reinterpret_cast<const uint32_t*>(w[i] + static_cast<int64_t>(u) * kMxUnitBytes + 4 * kMxTileBytes + lane * 4);
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const int k0 = u * kMxUnitCols + t * 128;
      if (k0 >= p.K) break;
      uint4 wv[NT];
#pragma unroll
      for (int i = 0; i < NT; ++i)
        wv[i] = *reinterpret_cast<const uint4*>(w[i] + static_cast<int64_t>(u) * kMxUnitBytes + t * kMxTileBytes + lane * 16);
      if constexpr (kMx8) {
        // x: lane (row, g) takes columns 16 g .. and 64 + 16 g .., scale of block g; past the last column, zeros
        i32x8 xv[MT];
        uint32_t xs[MT];
        const int ka = k0 + 16 * g, kb = ka + 64;
#pragma unroll
        for (int j = 0; j < MT; ++j) {
          const uint8_t* x = static_cast<const uint8_t*>(p.x) + row[j] * p.x_stride;
          uint4 a = make_uint4(0, 0, 0, 0), b = a;
          if (ka < p.K) a = *reinterpret_cast<const uint4*>(x + ka);
          if (kb < p.K) b = *reinterpret_cast<const uint4*>(x + kb);
          xv[j] = i32x8{(int)a.x, (int)a.y, (int)a.z, (int)a.w, (int)b.x, (int)b.y, (int)b.z, (int)b.w};
          xs[j] = k0 + 32 * g < p.K ? p.xs[row[j] * p.xs_stride + (k0 >> 5) + g] : 0u;
        }
#pragma unroll
        for (int i = 0; i < NT; ++i) {
          const i32x8 a = {(int)wv[i].x, (int)wv[i].y, (int)wv[i].z, (int)wv[i].w, 0, 0, 0, 0};
#pragma unroll
          for (int j = 0; j < MT; ++j)
            acc[i][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, xv[j], acc[i][j], 4, 0, 0,
                                                                         (ws[i] >> (8 * t)) & 0xffu, 0, xs[j]);
        }
      } else {
        const int k = k0 + 32 * g;
#pragma unroll
        for (int s = 0; s < 4; ++s) {
          uint4 xv[MT];
#pragma unroll
          for (int j = 0; j < MT; ++j) {
            xv[j] = make_uint4(0, 0, 0, 0);
            if (k < p.K) xv[j] = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p.x) + row[j] * p.x_stride + k + 8 * s);
          }
#pragma unroll
          for (int i = 0; i < NT; ++i) {
            const uint32_t c = s == 0 ? wv[i].x : s == 1 ? wv[i].y : s == 2 ? wv[i].z : wv[i].w;
            const uint4 a = e2m1_to_bf16(c, e8m0(ws[i], t));
#pragma unroll
            for (int j = 0; j < MT; ++j) acc[i][j] = mfma_bf16(a, xv[j], acc[i][j]);
          }
        }
      }
    }
  }
#pragma unroll
  for (int i = 0; i < NT; ++i) {
    if (i > 0) __syncthreads();
#pragma unroll
    for (int j = 0; j < MT; ++j) part[wave][j][lane] = acc[i][j];
    __syncthreads();
    const int j = threadIdx.x >> 6;
    const int n = (nt0 + i) * 16 + 4 * g, m = m0 + 16 * j + r;
    if (j < MT && m < p.M) {
      f32x4 s = part[0][j][lane];
#pragma unroll
      for (int v = 1; v < kWaves; ++v) s += part[v][j][lane];
      uint16_t* out = p.out + m * p.out_stride;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (n + e < p.N) out[n + e] = f32_to_bf16_bits(s[e] + (p.bias ? bf16_bits_to_f32(p.bias[n + e]) : 0.f));
    }
  }
}

template <bool kMx8, int MT>
void launch_rows(const LinearParams& p, hipStream_t s, int nt) {
  const int tiles = (p.N + 15) / 16;
  const dim3 grid(static_cast<unsigned>((tiles + nt - 1) / nt), static_cast<unsigned>((p.M + 16 * MT - 1) / (16 * MT)));
  if (nt == 4)
    mx4_rows_kernel<kMx8, MT, 4><<<grid, kWaves * 64, 0, s>>>(p);
  else if (nt == 2)
    mx4_rows_kernel<kMx8, MT, 2><<<grid, kWaves * 64, 0, s>>>(p);
  else
    mx4_rows_kernel<kMx8, MT, 1><<<grid, kWaves * 64, 0, s>>>(p);
}

template <bool kMx8>
int32_t launch(const LinearParams& p, hipStream_t s) {
  const int cus = device_cu_count();
  const int tiles = (p.N + 15) / 16;
  const int nt = tiles >= 4 * cus ? 4 : tiles >= 2 * cus ? 2 : 1;
  switch (std::min(4, (p.M + 15) / 16)) {
    case 1: launch_rows<kMx8, 1>(p, s, nt); break;
    case 2: launch_rows<kMx8, 2>(p, s, nt); break;
    case 3: launch_rows<kMx8, 3>(p, s, nt); break;
    default: launch_rows<kMx8, 4>(p, s, nt);
  }
  return check_launch("lkv_mx4_linear");
}

// ---- packing (off the path) ----

// Lane l of tile t of a unit: its 16 code bytes and its scale byte.  Rows and columns past the matrix: zeros.
struct PackItem {
  int64_t unit;
  int t, lane, n, k;
};

__device__ inline bool pack_item(int64_t id, int32_t units, int32_t N, int32_t K, PackItem& it) {
  it.lane = id & 63;
  it.t = (id >> 6) & 3;
  it.unit = id >> 8;
  it.n = static_cast<int>(it.unit / units) * 16 + (it.lane & 15);
  it.k = static_cast<int>(it.unit % units) * kMxUnitCols + it.t * 128 + 32 * (it.lane >> 4);
  return it.n < N && it.k < K;
}

__device__ inline void pack_store(uint8_t* out, const PackItem& it, uint4 codes, uint8_t scale) {
  uint8_t* unit = out + it.unit * kMxUnitBytes;
  *reinterpret_cast<uint4*>(unit + it.t * kMxTileBytes + it.lane * 16) = codes;
  unit[4 * kMxTileBytes + it.lane * 4 + it.t] = scale;
}

__global__ __launch_bounds__(256) void mx4_pack_kernel(const uint8_t* codes, int64_t c_stride, const uint8_t* scales,
                                                       int64_t s_stride, uint8_t* out, int32_t N, int32_t K, int32_t units,
                                                       int64_t items) {
  for (int64_t id = blockIdx.x * int64_t{256} + threadIdx.x; id < items; id += gridDim.x * int64_t{256}) {
    PackItem it;
    uint32_t v[4] = {0, 0, 0, 0};
    uint8_t s = 0;
    if (pack_item(id, units, N, K, it)) {
      const uint8_t* c = codes + it.n * c_stride + it.k / 2;
      for (int b = 0; b < 16; ++b) v[b >> 2] |= static_cast<uint32_t>(c[b]) << (8 * (b & 3));
      s = scales[it.n * s_stride + it.k / 32];
    }
    pack_store(out, it, make_uint4(v[0], v[1], v[2], v[3]), s);
  }
}

// A block's scale and codes from bf16: exponent of the maximum minus 2, one more where its mantissa passes 1.5;
// nearest code, ties to the even one.  A block with an infinity or NaN has the NaN scale.
__global__ __launch_bounds__(256) void mx4_quantize_kernel(const uint16_t* w, int64_t w_stride, uint8_t* out, int32_t N,
                                                           int32_t K, int32_t units, int64_t items) {
  for (int64_t id = blockIdx.x * int64_t{256} + threadIdx.x; id < items; id += gridDim.x * int64_t{256}) {
    PackItem it;
    uint32_t v[4] = {0, 0, 0, 0};
    uint8_t s = 0;
    if (pack_item(id, units, N, K, it)) {
      const uint16_t* x = w + it.n * w_stride + it.k;
      uint32_t amax = 0;  // of the bits without the sign: their order is the values'
      for (int b = 0; b < 32; ++b) amax = max(amax, x[b] & 0x7fffu);
      if (amax >= 0x7f80u) {
        s = 255;
      } else if (amax > 0) {
        int ex = static_cast<int>(amax >> 7), mant = amax & 0x7f;
        if (ex == 0) {  // below bf16's normal range: value mant * 2^-133
          const int top = 31 - __clz(mant);
          ex = top - 6;
          mant = (mant << (7 - top)) & 0x7f;
        }
        const int e = max(0, ex - 2 + (mant > 0x40));
        s = static_cast<uint8_t>(e);
        for (int b = 0; b < 32; ++b) {
          const float a = ldexpf(fabsf(bf16_bits_to_f32(x[b])), 127 - e);
          const uint32_t code = (a > 0.25f) + (a >= 0.75f) + (a > 1.25f) + (a >= 1.75f) + (a > 2.5f) + (a >= 3.5f) + (a > 5.f);
          v[b >> 3] |= (code | (x[b] >> 15) << 3) << (4 * (b & 7));
        }
      }
    }
    pack_store(out, it, make_uint4(v[0], v[1], v[2], v[3]), s);
  }
}

__global__ __launch_bounds__(256) void mx4_unpack_kernel(const uint8_t* w, uint16_t* out, int64_t o_stride, int32_t N,
                                                         int32_t K, int32_t units, int64_t items) {
  for (int64_t id = blockIdx.x * int64_t{256} + threadIdx.x; id < items; id += gridDim.x * int64_t{256}) {
    PackItem it;
    if (!pack_item(id, units, N, K, it)) continue;
    const uint8_t* unit = w + it.unit * kMxUnitBytes;
    const uint4 c = *reinterpret_cast<const uint4*>(unit + it.t * kMxTileBytes + it.lane * 16);
    const float s = e8m0(unit[4 * kMxTileBytes + it.lane * 4 + it.t], 0);
    uint4* o = reinterpret_cast<uint4*>(out + it.n * o_stride + it.k);
    o[0] = e2m1_to_bf16(c.x, s);
    o[1] = e2m1_to_bf16(c.y, s);
    o[2] = e2m1_to_bf16(c.z, s);
    o[3] = e2m1_to_bf16(c.w, s);
  }
}

int64_t pack_items(int32_t N, int32_t K) { return static_cast<int64_t>((N + 15) / 16) * mx4_units(K) * 256; }

unsigned pack_grid(int64_t items) { return static_cast<unsigned>(std::min<int64_t>((items + 255) / 256, 1 << 20)); }

uintptr_t bits(const void* p) { return reinterpret_cast<uintptr_t>(p); }

}  // namespace
}  // namespace lkv

#define LKV_REQUIRE_MX4_SHAPE(n, k)                                                                              \
  LKV_REQUIRE((n) > 0 && (n) <= (1 << 24) && (k) > 0 && (k) <= (1 << 24) && (k) % 32 == 0,                       \
              "an MX4 weight has 1 to 2^24 rows and a positive multiple of 32 columns up to 2^24, got %d x %d", n, k)

extern "C" int64_t lkv_mx4_weight_bytes(int32_t n, int32_t k) {
  if (n <= 0 || k <= 0) return 0;
  return static_cast<int64_t>((n + 15) / 16) * lkv::mx4_units(k) * lkv::kMxUnitBytes;
}

extern "C" int32_t lkv_mx4_pack(const void* codes, int64_t code_stride, const void* scales, int64_t scale_stride,
                                int32_t n, int32_t k, void* weight, lkv_stream_t stream) {
  using namespace lkv;
  LKV_REQUIRE(codes != nullptr && scales != nullptr && weight != nullptr, "null codes/scales/weight");
  LKV_REQUIRE_MX4_SHAPE(n, k);
  LKV_REQUIRE((bits(weight) & 15) == 0, "weight must be 16-byte aligned");
  const int64_t items = pack_items(n, k);
  mx4_pack_kernel<<<pack_grid(items), 256, 0, as_stream(stream)>>>(
      static_cast<const uint8_t*>(codes), code_stride, static_cast<const uint8_t*>(scales), scale_stride,
      static_cast<uint8_t*>(weight), n, k, static_cast<int32_t>(mx4_units(k)), items);
  return check_launch("lkv_mx4_pack");
}

extern "C" int32_t lkv_mx4_quantize(const void* src, int64_t src_stride, int32_t n, int32_t k, void* weight,
                                    lkv_stream_t stream) {
  using namespace lkv;
  LKV_REQUIRE(src != nullptr && weight != nullptr, "null src/weight");
  LKV_REQUIRE_MX4_SHAPE(n, k);
  LKV_REQUIRE((bits(weight) & 15) == 0 && (bits(src) & 1) == 0, "weight must be 16-byte aligned");
  const int64_t items = pack_items(n, k);
  mx4_quantize_kernel<<<pack_grid(items), 256, 0, as_stream(stream)>>>(static_cast<const uint16_t*>(src), src_stride,
                                                                      static_cast<uint8_t*>(weight), n, k,
                                                                      static_cast<int32_t>(mx4_units(k)), items);
  return check_launch("lkv_mx4_quantize");
}

extern "C" int32_t lkv_mx4_unpack(const void* weight, int32_t n, int32_t k, void* out, int64_t out_stride,
                                  lkv_stream_t stream) {
  using namespace lkv;
  LKV_REQUIRE(weight != nullptr && out != nullptr, "null weight/out");
  LKV_REQUIRE_MX4_SHAPE(n, k);
  LKV_REQUIRE(((bits(weight) | bits(out)) & 15) == 0 && out_stride % 8 == 0, "rows must be 16-byte aligned");
  const int64_t items = pack_items(n, k);
  mx4_unpack_kernel<<<pack_grid(items), 256, 0, as_stream(stream)>>>(static_cast<const uint8_t*>(weight),
                                                                    static_cast<uint16_t*>(out), out_stride, n, k,
                                                                    static_cast<int32_t>(mx4_units(k)), items);
  return check_launch("lkv_mx4_unpack");
}

extern "C" int32_t lkv_mx4_linear(const lkv_mx4_linear_args* a, lkv_stream_t stream) {
  using namespace lkv;
  LKV_REQUIRE(a != nullptr, "null args");
  LKV_REQUIRE(a->struct_size == static_cast<int32_t>(sizeof(lkv_mx4_linear_args)),
              "lkv_mx4_linear_args size mismatch (caller %d, library %d)", a->struct_size,
              static_cast<int32_t>(sizeof(lkv_mx4_linear_args)));
  LKV_REQUIRE(a->x_format == LKV_X_BF16 || a->x_format == LKV_X_MX8, "x_format must be LKV_X_BF16 or LKV_X_MX8, got %d",
              a->x_format);
  const bool mx8 = a->x_format == LKV_X_MX8;
  LKV_REQUIRE(a->rows >= 0 && a->rows <= (1 << 20), "rows must be in [0, 2^20], got %d", a->rows);
  LKV_REQUIRE_MX4_SHAPE(a->out_features, a->in_features);
  LKV_REQUIRE(a->x != nullptr && a->weight != nullptr && a->out != nullptr, "null x/weight/out");
  LKV_REQUIRE(mx8 == (a->x_scales != nullptr), "x_scales belong to MX8 rows, and they need them");
  LKV_REQUIRE(((bits(a->x) | bits(a->weight)) & 15) == 0 && ((bits(a->out) | bits(a->bias)) & 1) == 0,
              "x and weight must be 16-byte aligned");
  LKV_REQUIRE(a->x_stride % (mx8 ? 16 : 8) == 0, "x rows must be 16-byte aligned");
  if (a->rows == 0) return LKV_OK;
  LinearParams p;
  p.w = static_cast<const uint8_t*>(a->weight);
  p.x = a->x;
  p.x_stride = a->x_stride;
  p.xs = static_cast<const uint8_t*>(a->x_scales);
  p.xs_stride = a->x_scale_stride;
  p.bias = static_cast<const uint16_t*>(a->bias);
  p.out = static_cast<uint16_t*>(a->out);
  p.out_stride = a->out_stride;
  p.M = a->rows;
  p.N = a->out_features;
  p.K = a->in_features;
  p.units = static_cast<int32_t>(mx4_units(a->in_features));
  return mx8 ? launch<true>(p, as_stream(stream)) : launch<false>(p, as_stream(stream));
}
