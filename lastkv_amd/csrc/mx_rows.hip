// MX8 rows (e4m3 values, one e8m0 scale per 32): RMSNorm with the residual's addition and SwiGLU writing them, and
// their values in bf16 again.
#include <algorithm>

#include "mx.h"
#include "runtime.h"

namespace lkv {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxHidden = 16384;
constexpr int kMaxChunks = kMaxHidden / (kThreads * 8);

struct NormParams {
  const uint16_t* x;
  int64_t x_stride;
  uint16_t* residual;
  int64_t res_stride;
  const uint16_t* w;
  uint8_t* out;
  int64_t out_stride;
  uint8_t* scales;
  int64_t scale_stride;
  double eps;
  int32_t hidden;
};

__device__ inline void unpack8(uint4 u, float (&f)[8]) {
  f[0] = bf16_lo(u.x);
  f[1] = bf16_hi(u.x);
  f[2] = bf16_lo(u.y);
  f[3] = bf16_hi(u.y);
  f[4] = bf16_lo(u.z);
  f[5] = bf16_hi(u.z);
  f[6] = bf16_lo(u.w);
  f[7] = bf16_hi(u.w);
}

__device__ inline uint4 pack8(const float (&f)[8]) {
  return make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]), pack_bf16x2(f[6], f[7]));
}

// One workgroup per row; thread t owns the 8-element chunks t, t + 256, ... (kChunks of them).  With kAdd the row is
// residual := bf16(residual + x) first.  y = w * (row * r), r = 1 / sqrt(sum(row^2) / hidden + eps) with the sum and r in 64
// bits (no order of the sum then shows in a row's output, and no row's squares leave the range).
// Bound by HBM: every load is issued before the first use, with no branch between them (a chunk past the row rereads the
// last one); x and the residual are read once and take non-temporal accesses, as in lkv_rmsnorm.  4096 rows of 4096 with a
// residual: 21.8 us, 5.4 TB/s (lkv_rmsnorm, bf16 out, 22.7; the outputs all in 64 bits 32); one row 2.9.
template <bool kAdd, int kChunks>
__global__ __launch_bounds__(kThreads) void rmsnorm_mx8_kernel(const NormParams p) {
  __shared__ double part[kThreads / 64];
  const int row = blockIdx.x;
  const int chunks = p.hidden >> 3;
  const uint4* x = reinterpret_cast<const uint4*>(p.x + row * p.x_stride);
  uint4* res = kAdd ? reinterpret_cast<uint4*>(p.residual + row * p.res_stride) : nullptr;
  const uint4* w = reinterpret_cast<const uint4*>(p.w);
  uint4 xv[kChunks], rv[kChunks], wv[kChunks];
#pragma unroll
  for (int k = 0; k < kChunks; ++k) {
    const int c = min(static_cast<int>(threadIdx.x) + k * kThreads, chunks - 1);
    xv[k] = load_nt(x + c);
    if (kAdd) rv[k] = load_nt(res + c);
  }
#pragma unroll
  for (int k = 0; k < kChunks; ++k) wv[k] = w[min(static_cast<int>(threadIdx.x) + k * kThreads, chunks - 1)];
  double ss = 0.;
#pragma unroll
  for (int k = 0; k < kChunks; ++k) {
    const int c = threadIdx.x + k * kThreads;
    if (c < chunks) {
      float v[8];
      unpack8(xv[k], v);
      if (kAdd) {
        float r[8];
        unpack8(rv[k], r);
#pragma unroll
        for (int j = 0; j < 8; ++j) r[j] += v[j];
        xv[k] = pack8(r);
        __builtin_nontemporal_store(__builtin_bit_cast(u32x4, xv[k]), reinterpret_cast<u32x4*>(res + c));
        unpack8(xv[k], v);
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) ss = __builtin_fma(static_cast<double>(v[j]), static_cast<double>(v[j]), ss);
    }
  }
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) ss += __shfl_xor(ss, off);
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = ss;
  __syncthreads();
  const double total = (part[0] + part[1]) + (part[2] + part[3]);
  const double r = 1. / sqrt(total / p.hidden + p.eps);
  const float rf = static_cast<float>(r);
#pragma unroll
  for (int k = 0; k < kChunks; ++k) {
    const int c = threadIdx.x + k * kThreads;
    if (c < chunks) {  // (a block's four chunks are all inside the row or all outside)
      float h[8], wf[8], y[8];
      unpack8(xv[k], h);
      unpack8(wv[k], wf);
#pragma unroll
      for (int j = 0; j < 8; ++j) y[j] = wf[j] * (h[j] * rf);  // (three roundings: within 2^-22)
      // ... where h rf stays in fp32's normal range.  Below it another 2^-150 |w| are missing, up to 2^-43 of a block's
      // maximum for |w| <= 2^10 (that is at least 2^-97), 2^-24 of what does not round to zero; larger weights take 64 bits.
      const float wmax = fmax_nan(fmax3_nan(fmax3_nan(fmax3_nan(fabsf(wf[0]), fabsf(wf[1]), fabsf(wf[2])), fabsf(wf[3]), fabsf(wf[4])),
                                            fabsf(wf[5]), fabsf(wf[6])), fabsf(wf[7]));
      if (wmax > 0x1p10f) y[0] = __uint_as_float(0x7fc00000u);
      int byte;
      const uint2 q = quantize_e4m3(y, byte, [&](double(&d)[8]) {
#pragma unroll
        for (int j = 0; j < 8; ++j) d[j] = static_cast<double>(wf[j]) * (static_cast<double>(h[j]) * r);
      });
      reinterpret_cast<uint2*>(p.out + row * p.out_stride)[c] = q;
      if ((c & 3) == 0) p.scales[row * p.scale_stride + (c >> 2)] = static_cast<uint8_t>(byte);
    }
  }
}

// g / (1 + e^-g) for -80 <= g within 2^-21.4: v_exp_f32 and v_rcp_f32 are off by one unit in the last place (2^-23), the
// product with log2(e) is carried in two parts, the reciprocal takes one Newton step.  (Above 80 the sum is 1.)
__device__ inline float silu(float g) {
  const float x = -fminf(g, 80.f);
  const float hi = x * kLog2e, lo = __builtin_fmaf(x, kLog2e, -hi);
  const float e = fast_exp2(hi);
  const float d = 1.f + __builtin_fmaf(e, lo * kLn2, e);
  const float r = __builtin_amdgcn_rcpf(d);
  return g * __builtin_fmaf(__builtin_fmaf(-d, r, 1.f), r, r);
}

// y = silu(gate) * up; grid (column groups, rows), one 8-element chunk per thread.  Bound by HBM: 4096 rows of 14336 in
// 50.5 us, 5.9 TB/s (lkv_silu_mul, bf16 out, 52.4; in 64 bits 138); 32 rows 4.3.
__global__ __launch_bounds__(256) void silu_mul_mx8_kernel(const uint16_t* gate, int64_t g_stride, const uint16_t* up,
                                                           int64_t u_stride, uint8_t* out, int64_t o_stride,
                                                           uint8_t* scales, int64_t s_stride, int32_t rows,
                                                           int32_t width) {
  const int c = blockIdx.x * 256 + threadIdx.x;
  if (c >= width >> 3) return;
  for (int64_t row = blockIdx.y; row < rows; row += gridDim.y) {
    float g[8], u[8], y[8];
    unpack8(load_nt(reinterpret_cast<const uint4*>(gate + row * g_stride) + c), g);
    unpack8(load_nt(reinterpret_cast<const uint4*>(up + row * u_stride) + c), u);
    float least = g[0];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      y[j] = silu(g[j]) * u[j];
      least = fminf(least, g[j]);
    }
    if (least < -80.f) y[0] = __uint_as_float(0x7fc00000u);  // e^-g leaves the range that silu() takes: in 64 bits
    int byte;
    const uint2 q = quantize_e4m3(y, byte, [&](double(&d)[8]) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const double x = g[j];
        d[j] = x / (1. + exp(-x)) * static_cast<double>(u[j]);
      }
    });
    reinterpret_cast<uint2*>(out + row * o_stride)[c] = q;
    if ((c & 3) == 0) scales[row * s_stride + (c >> 2)] = static_cast<uint8_t>(byte);
  }
}

// bf16(e4m3 * 2^(e - 127)), 8 values per thread: HBM, 4096 rows of 14336 in 26.8 us, 6.6 TB/s.  (An output below bf16's
// normal range rounds, one above it is infinite.)
__global__ __launch_bounds__(256) void mx8_unpack_kernel(const uint8_t* data, int64_t d_stride, const uint8_t* scales,
                                                         int64_t s_stride, uint16_t* out, int64_t o_stride, int32_t rows,
                                                         int32_t width) {
  const int c = blockIdx.x * 256 + threadIdx.x;
  if (c >= width >> 3) return;
  for (int64_t row = blockIdx.y; row < rows; row += gridDim.y) {
    const uint2 q = reinterpret_cast<const uint2*>(data + row * d_stride)[c];
    const uint32_t e = scales[row * s_stride + (c >> 2)];
    const float s = e == 0 ? __uint_as_float(0x00400000u) : e == 255 ? __uint_as_float(0x7fc00000u) : __uint_as_float(e << 23);
    float v[8];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const auto a = __builtin_amdgcn_cvt_pk_f32_fp8(h ? q.y : q.x, false);
      const auto b = __builtin_amdgcn_cvt_pk_f32_fp8(h ? q.y : q.x, true);
      v[4 * h] = a[0] * s;
      v[4 * h + 1] = a[1] * s;
      v[4 * h + 2] = b[0] * s;
      v[4 * h + 3] = b[1] * s;
    }
    reinterpret_cast<uint4*>(out + row * o_stride)[c] = pack8(v);
  }
}

constexpr int32_t kMaxNormRows = 1 << 23;  // of a launch: a grid has fewer than 2^32 threads

template <bool kAdd>
void launch_norm(NormParams p, int32_t rows, hipStream_t s) {
  const int chunks = (p.hidden + kThreads * 8 - 1) / (kThreads * 8);
  while (rows > 0) {
    const int32_t n = std::min(rows, kMaxNormRows);
    if (chunks <= 1)
      rmsnorm_mx8_kernel<kAdd, 1><<<n, kThreads, 0, s>>>(p);
    else if (chunks <= 2)
      rmsnorm_mx8_kernel<kAdd, 2><<<n, kThreads, 0, s>>>(p);
    else if (chunks <= 4)
      rmsnorm_mx8_kernel<kAdd, 4><<<n, kThreads, 0, s>>>(p);
    else
      rmsnorm_mx8_kernel<kAdd, kMaxChunks><<<n, kThreads, 0, s>>>(p);
    rows -= n;
    p.x += n * p.x_stride;
    if (kAdd) p.residual += n * p.res_stride;
    p.out += n * p.out_stride;
    p.scales += n * p.scale_stride;
  }
}

dim3 row_grid(int32_t rows, int32_t width) {
  return dim3(static_cast<unsigned>((width / 8 + 255) / 256), static_cast<unsigned>(std::min(rows, 65535)));
}

uintptr_t bits(const void* p) { return reinterpret_cast<uintptr_t>(p); }

}  // namespace
}  // namespace lkv

extern "C" int32_t lkv_rmsnorm_mx8(const lkv_rmsnorm_mx8_args* a, lkv_stream_t stream) {
  using namespace lkv;
  LKV_REQUIRE(a != nullptr, "null args");
  LKV_REQUIRE(a->struct_size == static_cast<int32_t>(sizeof(lkv_rmsnorm_mx8_args)),
              "lkv_rmsnorm_mx8_args size mismatch (caller %d, library %d)", a->struct_size,
              static_cast<int32_t>(sizeof(lkv_rmsnorm_mx8_args)));
  LKV_REQUIRE(a->rows >= 0, "rows must be non-negative");
  LKV_REQUIRE(a->hidden > 0 && a->hidden % kMxBlock == 0 && a->hidden <= kMaxHidden,
              "hidden must be a positive multiple of 32 up to %d, got %d", kMaxHidden, a->hidden);
  LKV_REQUIRE(a->x != nullptr && a->weight != nullptr && a->out != nullptr && a->scales != nullptr,
              "null x/weight/out/scales");
  LKV_REQUIRE(((bits(a->x) | bits(a->weight) | bits(a->residual)) & 15) == 0 && (bits(a->out) & 7) == 0,
              "rows must be 16-byte aligned (8-bit ones 8)");
  LKV_REQUIRE((a->x_stride | a->out_stride | a->residual_stride) % 8 == 0, "row strides must be multiples of 8 elements");
  LKV_REQUIRE(a->rows <= 1 || (a->out_stride >= a->hidden && a->scale_stride >= a->hidden / kMxBlock &&
                               (a->residual == nullptr || a->residual_stride >= a->hidden)),
              "rows of residual, out and scales must not overlap");
  if (a->rows == 0) return LKV_OK;
  NormParams p;
  p.x = static_cast<const uint16_t*>(a->x);
  p.x_stride = a->x_stride;
  p.residual = static_cast<uint16_t*>(a->residual);
  p.res_stride = a->residual_stride;
  p.w = static_cast<const uint16_t*>(a->weight);
  p.out = static_cast<uint8_t*>(a->out);
  p.out_stride = a->out_stride;
  p.scales = static_cast<uint8_t*>(a->scales);
  p.scale_stride = a->scale_stride;
  p.hidden = a->hidden;
  p.eps = a->eps;
  hipStream_t s = as_stream(stream);
  if (a->residual != nullptr)
    launch_norm<true>(p, a->rows, s);
  else
    launch_norm<false>(p, a->rows, s);
  return check_launch("lkv_rmsnorm_mx8");
}

extern "C" int32_t lkv_silu_mul_mx8(const void* gate, int64_t gate_stride, const void* up, int64_t up_stride, void* out,
                                    int64_t out_stride, void* scales, int64_t scale_stride, int32_t rows, int32_t width,
                                    lkv_stream_t stream) {
  using namespace lkv;
  LKV_REQUIRE(gate != nullptr && up != nullptr && out != nullptr && scales != nullptr, "null gate/up/out/scales");
  LKV_REQUIRE(rows >= 0 && width > 0 && width % kMxBlock == 0, "width must be a positive multiple of 32");
  LKV_REQUIRE(((bits(gate) | bits(up)) & 15) == 0 && (bits(out) & 7) == 0, "rows must be 16-byte aligned (8-bit ones 8)");
  LKV_REQUIRE((gate_stride | up_stride | out_stride) % 8 == 0, "row strides must be multiples of 8 elements");
  LKV_REQUIRE(rows <= 1 || (out_stride >= width && scale_stride >= width / kMxBlock), "rows of out and scales must not overlap");
  if (rows == 0) return LKV_OK;
  silu_mul_mx8_kernel<<<row_grid(rows, width), 256, 0, as_stream(stream)>>>(
      static_cast<const uint16_t*>(gate), gate_stride, static_cast<const uint16_t*>(up), up_stride,
      static_cast<uint8_t*>(out), out_stride, static_cast<uint8_t*>(scales), scale_stride, rows, width);
  return check_launch("lkv_silu_mul_mx8");
}

extern "C" int32_t lkv_mx8_unpack(const void* data, int64_t data_stride, const void* scales, int64_t scale_stride,
                                  void* out, int64_t out_stride, int32_t rows, int32_t width, lkv_stream_t stream) {
  using namespace lkv;
  LKV_REQUIRE(data != nullptr && scales != nullptr && out != nullptr, "null data/scales/out");
  LKV_REQUIRE(rows >= 0 && width > 0 && width % kMxBlock == 0, "width must be a positive multiple of 32");
  LKV_REQUIRE((bits(out) & 15) == 0 && (bits(data) & 7) == 0, "rows must be 16-byte aligned (8-bit ones 8)");
  LKV_REQUIRE((data_stride | out_stride) % 8 == 0, "row strides must be multiples of 8 elements");
  LKV_REQUIRE(rows <= 1 || out_stride >= width, "out rows must not overlap");
  if (rows == 0) return LKV_OK;
  mx8_unpack_kernel<<<row_grid(rows, width), 256, 0, as_stream(stream)>>>(
      static_cast<const uint8_t*>(data), data_stride, static_cast<const uint8_t*>(scales), scale_stride,
      static_cast<uint16_t*>(out), out_stride, rows, width);
  return check_launch("lkv_mx8_unpack");
}
