// Conversion of bf16 pages (the tiled layout of common.h) to 8-bit pages and back to rows.
//
// Quantising a block: amax = max|x| over its valid tokens, E the smallest integer >= -127 with amax <= 448 * 2^E, codes
// e4m3(x * 2^-E) rounded to nearest even.  Bound by memory: 2 bytes read and 1 written a value.  One workgroup a (block, kv head,
// sequence) takes K and V: a thread holds 16 values of each (two bf16 operands of its lane, 16 bytes of the 8-bit
// block), so every load and store is 16 bytes a lane and nothing but the two maxima passes through LDS.
#include "kv8.h"

namespace lkv {

int32_t kv8_pool(const lkv_kv8_pool* a, const char* name, Kv8Pool& p) {
  LKV_REQUIRE(a != nullptr, "null %s", name);
  LKV_REQUIRE(a->struct_size == static_cast<int32_t>(sizeof(lkv_kv8_pool)), "lkv_kv8_pool size mismatch (caller %d, library %d)",
              a->struct_size, static_cast<int32_t>(sizeof(lkv_kv8_pool)));
  LKV_REQUIRE(a->k && a->v && a->k_scales && a->v_scales, "%s: null tensor", name);
  LKV_REQUIRE(a->num_pages > 0 && a->heads > 0, "%s: an 8-bit pool needs pages and heads", name);
  LKV_REQUIRE(((reinterpret_cast<uintptr_t>(a->k) | reinterpret_cast<uintptr_t>(a->v)) & 15) == 0,
              "%s: 8-bit pools must be 16-byte aligned", name);
  LKV_REQUIRE(a->page_stride >= kKv8Block && a->page_stride % 16 == 0 && a->head_stride >= 0 && a->head_stride % 16 == 0,
              "%s: strides of an 8-bit pool must be multiples of 16 bytes, a page at least 4096", name);
  // (the attention reads scales by words)
  LKV_REQUIRE(((reinterpret_cast<uintptr_t>(a->k_scales) | reinterpret_cast<uintptr_t>(a->v_scales)) & 3) == 0 &&
                  a->scale_head_stride % 4 == 0 && a->scale_head_stride >= a->num_pages,
              "%s: scales of an 8-bit pool must be 4-byte aligned, scale_head_stride a multiple of 4 that holds the pages", name);
  p.k = static_cast<const uint8_t*>(a->k);
  p.v = static_cast<const uint8_t*>(a->v);
  p.ks = static_cast<const uint8_t*>(a->k_scales);
  p.vs = static_cast<const uint8_t*>(a->v_scales);
  p.page = a->page_stride;
  p.hs = a->head_stride;
  p.s_hs = a->scale_head_stride;
  p.pages = a->num_pages;
  return LKV_OK;
}

namespace {

// Calls over more bf16 values than this read non-temporally: 16 sequences of 8192 tokens (512 MiB), replayed, are quantised in 123 us
// (6.5 TB/s of reads and writes) so and in 164 with plain loads, unpacked in 144 and 148; calls of 1024 tokens each, which the caches
// hold, take plain loads (19.2 us quantised and 20.0 unpacked without, 16.8 and 17.0 with them).
constexpr int64_t kNtBytes = int64_t{384} << 20;

struct QuantizeParams {
  const uint16_t* k;
  const uint16_t* v;
  int64_t page, hs;
  int32_t pages;
  const int32_t* src_table;
  const int32_t* dst_table;
  int64_t src_ts, dst_ts;
  const int32_t* tokens;
  int32_t tokens_c, first;
  Kv8Pool dst;
};

__device__ inline uint32_t max_bits(uint4 x, uint32_t m) {
#pragma unroll
  for (const uint32_t w : {x.x, x.y, x.z, x.w}) m = max(max(m, w & 0x7fffu), (w >> 16) & 0x7fffu);
  return m;
}

template <int kCtrl>
__device__ inline uint32_t max_dpp(uint32_t x) {
  return max(x, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, x, kCtrl, 0xf, 0xf, true)));
}

// The greatest of the wave's, without LDS: within quads, the halves of a row, the row, then across rows.
__device__ inline uint32_t wave_max_bits(uint32_t x) {
  x = max_dpp<0x140>(max_dpp<0x141>(max_dpp<0x4e>(max_dpp<0xb1>(x))));
  const auto a = __builtin_amdgcn_permlane16_swap(x, x, false, false);
  x = max(a[0], a[1]);
  const auto c = __builtin_amdgcn_permlane32_swap(x, x, false, false);
  return max(c[0], c[1]);
}

template <bool kNt>
__device__ inline uint4 load16(const void* p) {
  return kNt ? load_nt(p) : *reinterpret_cast<const uint4*>(p);
}

// Two e4m3 codes of a packed bf16 pair times f, in the low or high half.
template <bool kHigh>
__device__ inline int code_pair(int old, uint32_t w, float f) {
  return __builtin_amdgcn_cvt_pk_fp8_f32(bf16_lo(w) * f, bf16_hi(w) * f, old, kHigh);
}

__device__ inline uint2 codes8(uint4 x, float f) {
  return make_uint2(code_pair<true>(code_pair<false>(0, x.x, f), x.y, f), code_pair<true>(code_pair<false>(0, x.z, f), x.w, f));
}

// The scale byte of a block whose greatest |x| has these bf16 bits: |x| = (1 + man / 128) 2^(exp - 127), and 448 = 1.75 * 2^8.
__device__ inline int scale_byte(uint32_t bits) {
  const int ex = static_cast<int>(bits >> 7);
  return ex == 255 ? 255 : max(0, ex - 8 + ((bits & 0x7fu) > 0x60u));
}

template <bool kNt>
__global__ __launch_bounds__(256) void kv8_quantize_kernel(const QuantizeParams p) {
  __shared__ uint32_t sm_max[2][4];
  const int b = blockIdx.z, h = blockIdx.y, j = p.first + blockIdx.x;
  const int total = p.tokens ? p.tokens[b] : p.tokens_c;
  const int valid = min(max(total, 0) - min(max(total, 0), j * kBlockTokens), kBlockTokens);
  if (valid <= 0) return;  // (workgroup-uniform)
  const int lane = threadIdx.x & 63, piece = threadIdx.x >> 6, n16 = lane & 15, g4 = lane >> 4;
  const int sp = min(max(p.src_table[b * p.src_ts + j], 0), p.pages - 1);
  const int dp = min(max(p.dst_table[b * p.dst_ts + j], 0), p.dst.pages - 1);
  const int64_t so = sp * p.page + h * p.hs;
  uint4 k[2], v[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    // K: piece = u * 2 + kp, operand kb = 2 kp + i; V: operand nb = 2 piece + i
    k[i] = load16<kNt>(p.k + so + (((piece >> 1) * 4 + (piece & 1) * 2 + i) * 16 + n16) * 32 + 8 * g4);
    v[i] = load16<kNt>(p.v + so + (16 * (2 * piece + i) + n16) * 32 + 8 * g4);
  }
  if (valid < kBlockTokens) {  // what lies past the sequence's end does not count and is stored as 0
    const int w = ((n16 >> 2) << 3) | ((piece >> 1) << 2) | (n16 & 3);  // this thread's K token
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      if (w >= valid) k[i] = make_uint4(0, 0, 0, 0);
      v[i] = keep_tokens(v[i], valid - 8 * g4);
    }
  }
  uint32_t mk = max_bits(k[1], max_bits(k[0], 0)), mv = max_bits(v[1], max_bits(v[0], 0));
  mk = wave_max_bits(mk);
  mv = wave_max_bits(mv);
  if (lane == 0) {
    sm_max[0][piece] = mk;
    sm_max[1][piece] = mv;
  }
  __syncthreads();
  mk = max(max(sm_max[0][0], sm_max[0][1]), max(sm_max[0][2], sm_max[0][3]));
  mv = max(max(sm_max[1][0], sm_max[1][1]), max(sm_max[1][2], sm_max[1][3]));
  const int ek = scale_byte(mk), ev = scale_byte(mv);
  // (2^(127 - e), e <= 247 for finite blocks; a NaN block's codes are 0)
  const float fk = ek == 255 ? 0.f : __uint_as_float(static_cast<uint32_t>(254 - ek) << 23);
  const float fv = ev == 255 ? 0.f : __uint_as_float(static_cast<uint32_t>(254 - ev) << 23);
  uint2 k0 = codes8(k[0], fk), k1 = codes8(k[1], fk), v0 = codes8(v[0], fv), v1 = codes8(v[1], fv);
  if (ek == 255) k0 = k1 = make_uint2(0, 0);
  if (ev == 255) v0 = v1 = make_uint2(0, 0);
  const int64_t at = dp * p.dst.page + h * p.dst.hs + threadIdx.x * 16;
  *reinterpret_cast<uint4*>(const_cast<uint8_t*>(p.dst.k) + at) = make_uint4(k0.x, k0.y, k1.x, k1.y);
  *reinterpret_cast<uint4*>(const_cast<uint8_t*>(p.dst.v) + at) = make_uint4(v0.x, v0.y, v1.x, v1.y);
  if (threadIdx.x == 0) {
    const_cast<uint8_t*>(p.dst.ks)[h * p.dst.s_hs + dp] = static_cast<uint8_t>(ek);
    const_cast<uint8_t*>(p.dst.vs)[h * p.dst.s_hs + dp] = static_cast<uint8_t>(ev);
  }
}

struct UnpackParams {
  Kv8Pool src;
  const int32_t* table;
  int64_t ts;
  uint16_t* k;
  uint16_t* v;
  int64_t ksb, ksh, kst, vsb, vsh, vst;
  int32_t token0, tokens;
};

// One workgroup a (block, kv head, sequence).  A thread's 16 K codes are 8 + 8 dims of one token, stored as they are; V
// (16 codes of two dims) turns through LDS into 16 dims of one token.
template <bool kNt>
__global__ __launch_bounds__(256) void kv8_unpack_kernel(const UnpackParams p) {
  __shared__ __align__(16) uint8_t sm[kBlockTokens][kHeadDim];
  const int b = blockIdx.z, h = blockIdx.y, j = (p.token0 >> 5) + blockIdx.x;
  const int lane = threadIdx.x & 63, piece = threadIdx.x >> 6, n16 = lane & 15, g4 = lane >> 4;
  const int page = min(max(p.table[b * p.ts + j], 0), p.src.pages - 1);
  const int64_t at = page * p.src.page + h * p.src.hs + threadIdx.x * 16;
  const uint4 k = load16<kNt>(p.src.k + at), v = load16<kNt>(p.src.v + at);
  const float sk = kv8_scale(p.src.ks[h * p.src.s_hs + page]), sv = kv8_scale(p.src.vs[h * p.src.s_hs + page]);
  const int t0 = j * kBlockTokens - p.token0;  // row of the block's token 0
  {
    const int t = t0 + (((n16 >> 2) << 3) | ((piece >> 1) << 2) | (n16 & 3));
    if (t >= 0 && t < p.tokens) {
      uint16_t* row = p.k + b * p.ksb + h * p.ksh + t * p.kst + (piece & 1) * 64 + 8 * g4;
      *reinterpret_cast<uint4*>(row) = kv8_to_bf16(k.x, k.y, sk);
      *reinterpret_cast<uint4*>(row + 32) = kv8_to_bf16(k.z, k.w, sk);
    }
  }
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 16; ++i)
    sm[8 * g4 + (i & 7)][32 * piece + 16 * (i >> 3) + n16] = static_cast<uint8_t>(w[i >> 2] >> (8 * (i & 3)));
  __syncthreads();
  const int tok = threadIdx.x >> 3, d0 = (threadIdx.x & 7) * 16, t = t0 + tok;
  if (t >= 0 && t < p.tokens) {
    const uint4 c = *reinterpret_cast<const uint4*>(&sm[tok][d0]);
    uint16_t* row = p.v + b * p.vsb + h * p.vsh + t * p.vst + d0;
    *reinterpret_cast<uint4*>(row) = kv8_to_bf16(c.x, c.y, sv);
    *reinterpret_cast<uint4*>(row + 8) = kv8_to_bf16(c.z, c.w, sv);
  }
}

}  // namespace
}  // namespace lkv

extern "C" int32_t lkv_kv8_quantize(const lkv_kv8_quantize_args* a, const lkv_kv8_pool* dst, lkv_stream_t stream) {
  using namespace lkv;
  LKV_REQUIRE(a != nullptr, "null args");
  LKV_REQUIRE(a->struct_size == static_cast<int32_t>(sizeof(lkv_kv8_quantize_args)),
              "lkv_kv8_quantize_args size mismatch (caller %d, library %d)", a->struct_size,
              static_cast<int32_t>(sizeof(lkv_kv8_quantize_args)));
  QuantizeParams p;
  if (const int32_t st = kv8_pool(dst, "dst", p.dst)) return st;
  LKV_REQUIRE(a->head_dim == kHeadDim, "head_dim must be 128, got %d", a->head_dim);
  LKV_REQUIRE(a->batch >= 0 && a->blocks >= 0 && a->first_block >= 0, "bad sizes");
  LKV_REQUIRE(a->heads == dst->heads, "the pools have %d and %d kv heads", a->heads, dst->heads);
  if (a->batch == 0 || a->blocks == 0) return LKV_OK;  // (empty tensors have no address)
  LKV_REQUIRE(a->src_k && a->src_v && a->src_table && a->dst_table, "null tensor");
  LKV_REQUIRE(a->src_num_pages > 0, "src_num_pages must be positive");
  LKV_REQUIRE(((reinterpret_cast<uintptr_t>(a->src_k) | reinterpret_cast<uintptr_t>(a->src_v)) & 15) == 0 &&
                  ((a->src_page_stride | a->src_head_stride) & 7) == 0,
              "source pages must be 16-byte aligned");
  LKV_REQUIRE(a->tokens != nullptr || a->tokens_const >= 0, "negative token count");
  const int64_t end = static_cast<int64_t>(a->first_block) + a->blocks;
  LKV_REQUIRE(end <= a->src_table_width && end <= a->dst_table_width,
              "blocks [%d, %lld) exceed the tables' %d and %d", a->first_block, static_cast<long long>(end),
              a->src_table_width, a->dst_table_width);
  LKV_REQUIRE(a->batch <= 65535 && a->heads <= 65535 && end < (1 << 24), "batch and heads must be <= 65535, blocks < 2^24");
  p.k = static_cast<const uint16_t*>(a->src_k);
  p.v = static_cast<const uint16_t*>(a->src_v);
  p.page = a->src_page_stride;
  p.hs = a->src_head_stride;
  p.pages = a->src_num_pages;
  p.src_table = a->src_table;
  p.dst_table = a->dst_table;
  p.src_ts = a->src_table_stride;
  p.dst_ts = a->dst_table_stride;
  p.tokens = a->tokens;
  p.tokens_c = a->tokens_const;
  p.first = a->first_block;
  const dim3 grid(a->blocks, a->heads, a->batch);
  if (static_cast<int64_t>(a->batch) * a->heads * a->blocks * kBlockElems * 4 > kNtBytes)
    kv8_quantize_kernel<true><<<grid, 256, 0, as_stream(stream)>>>(p);
  else
    kv8_quantize_kernel<false><<<grid, 256, 0, as_stream(stream)>>>(p);
  return check_launch("lkv_kv8_quantize");
}

extern "C" int32_t lkv_kv8_unpack(const lkv_kv8_pool* src, const int32_t* table, int64_t table_stride, int32_t table_width,
                                  int32_t batch, int32_t token0, int32_t tokens, void* k, int64_t k_stride_b,
                                  int64_t k_stride_h, int64_t k_stride_t, void* v, int64_t v_stride_b, int64_t v_stride_h,
                                  int64_t v_stride_t, lkv_stream_t stream) {
  using namespace lkv;
  UnpackParams p;
  if (const int32_t st = kv8_pool(src, "src", p.src)) return st;
  LKV_REQUIRE(batch >= 0 && token0 >= 0 && tokens >= 0, "bad sizes");
  const int64_t end = (static_cast<int64_t>(token0) + tokens + kBlockTokens - 1) / kBlockTokens;
  LKV_REQUIRE(end <= table_width, "tokens [%d, %lld) exceed the table's %d blocks", token0,
              static_cast<long long>(token0) + tokens, table_width);
  LKV_REQUIRE(((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & 15) == 0 &&
                  ((k_stride_b | k_stride_h | k_stride_t | v_stride_b | v_stride_h | v_stride_t) & 7) == 0,
              "rows must be 16-byte aligned");
  LKV_REQUIRE(batch <= 65535 && src->heads <= 65535 && end < (1 << 24), "batch and heads must be <= 65535, blocks < 2^24");
  if (batch == 0 || tokens == 0) return LKV_OK;  // (empty tensors have no address)
  LKV_REQUIRE(table && k && v, "null tensor");
  p.table = table;
  p.ts = table_stride;
  p.k = static_cast<uint16_t*>(k);
  p.v = static_cast<uint16_t*>(v);
  p.ksb = k_stride_b;
  p.ksh = k_stride_h;
  p.kst = k_stride_t;
  p.vsb = v_stride_b;
  p.vsh = v_stride_h;
  p.vst = v_stride_t;
  p.token0 = token0;
  p.tokens = tokens;
  const dim3 grid(static_cast<unsigned>(end - (token0 >> 5)), src->heads, batch);
  if (static_cast<int64_t>(batch) * src->heads * grid.x * kBlockElems * 4 > kNtBytes)
    kv8_unpack_kernel<true><<<grid, 256, 0, as_stream(stream)>>>(p);
  else
    kv8_unpack_kernel<false><<<grid, 256, 0, as_stream(stream)>>>(p);
  return check_launch("lkv_kv8_unpack");
}
