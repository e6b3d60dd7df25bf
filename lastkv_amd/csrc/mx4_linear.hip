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
  int32_t units, tile_stride;
  bool vector_out;  // output rows are 16-byte aligned
};

constexpr int kWaves = 8;
constexpr int kStepTiles = 2;                  // 128-column tiles that a wave loads at once
constexpr int kStepCols = 128 * kStepTiles;

// Byte t of a scale word as the exponent of a float (the converts read no other bits; 0 stands for 2^-127).
__device__ inline float e8m0(uint32_t word, int t) { return __uint_as_float(((word >> (8 * t)) & 0xffu) << 23); }

// Eight e2m1 codes of a word as scaled bf16 (exact: 2 significant bits, bf16's exponents).
__device__ inline uint4 e2m1_to_bf16(uint32_t codes, float scale) {
  return make_uint4(__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 0)),
                    __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 1)),
                    __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 2)),
                    __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 3)));
}

// Eight e4m3 values of two words as scaled bf16 (exact inside bf16's range).
__device__ inline uint4 e4m3_to_bf16(uint32_t a, uint32_t b, float scale) {
  return make_uint4(__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, scale, false)),
                    __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, scale, true)),
                    __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, scale, false)),
                    __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, scale, true)));
}

__device__ inline uint32_t word_of(const uint4& v, int j) { return j == 0 ? v.x : j == 1 ? v.y : j == 2 ? v.z : v.w; }

__device__ inline uint4 buffer_load16(__amdgpu_buffer_rsrc_t r, int offset, int scalar_offset = 0) {
  return __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(r, offset, scalar_offset, 0));
}

// 16 bytes of each lane to LDS at `dst` + 16 lane (dst the same for the wave), past the registers.
__device__ inline void buffer_to_lds16(__amdgpu_buffer_rsrc_t r, char* dst, int offset, int scalar_offset) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void*)dst, 16, offset, scalar_offset, 0, 0);
}

__device__ inline uint32_t lds_address(const void* p) {
  return static_cast<uint32_t>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) const char*)p));
}

// A wave's fragments of a tile (4 of codes, 2 of x), read and waited for in one piece of assembly: before an LDS read of its
// own the compiler waits for every load to LDS in flight, those of later tiles too.
template <int kXStep>
__device__ inline void read_mx8(uint32_t w, uint32_t lo, uint32_t hi, uint4 (&c)[4], uint4 (&l)[2], uint4 (&h)[2]) {
  asm volatile(
      "ds_read_b128 %0, %8\n ds_read_b128 %4, %9\n ds_read_b128 %6, %10\n"
      "ds_read_b128 %5, %9 offset:%c11\n ds_read_b128 %7, %10 offset:%c11\n"
      "ds_read_b128 %1, %8 offset:%c12\n ds_read_b128 %2, %8 offset:%c13\n ds_read_b128 %3, %8 offset:%c14\n"
      "s_waitcnt lgkmcnt(0)"
      : "=&v"(c[0]), "=&v"(c[1]), "=&v"(c[2]), "=&v"(c[3]), "=&v"(l[0]), "=&v"(l[1]), "=&v"(h[0]), "=&v"(h[1])
      : "v"(w), "v"(lo), "v"(hi), "n"(kXStep), "n"(kMxTileBytes), "n"(2 * kMxTileBytes), "n"(3 * kMxTileBytes)
      : "memory");
}

// Likewise the fragments of 4 tiles of bf16 rows, from where their four steps' chunks start.
template <int kXStep>
__device__ inline void read_bf16(const uint32_t (&x)[4], uint4 (&b)[4][4]) {
  asm volatile(
      "ds_read_b128 %0, %16\n ds_read_b128 %1, %16 offset:%c20\n ds_read_b128 %2, %16 offset:%c21\n ds_read_b128 %3, %16 offset:%c22\n"
      "ds_read_b128 %4, %17\n ds_read_b128 %5, %17 offset:%c20\n ds_read_b128 %6, %17 offset:%c21\n ds_read_b128 %7, %17 offset:%c22\n"
      "ds_read_b128 %8, %18\n ds_read_b128 %9, %18 offset:%c20\n ds_read_b128 %10, %18 offset:%c21\n ds_read_b128 %11, %18 offset:%c22\n"
      "ds_read_b128 %12, %19\n ds_read_b128 %13, %19 offset:%c20\n ds_read_b128 %14, %19 offset:%c21\n"
      "ds_read_b128 %15, %19 offset:%c22\n s_waitcnt lgkmcnt(0)"
      : "=&v"(b[0][0]), "=&v"(b[0][1]), "=&v"(b[0][2]), "=&v"(b[0][3]), "=&v"(b[1][0]), "=&v"(b[1][1]), "=&v"(b[1][2]),
        "=&v"(b[1][3]), "=&v"(b[2][0]), "=&v"(b[2][1]), "=&v"(b[2][2]), "=&v"(b[2][3]), "=&v"(b[3][0]), "=&v"(b[3][1]),
        "=&v"(b[3][2]), "=&v"(b[3][3])
      : "v"(x[0]), "v"(x[1]), "v"(x[2]), "v"(x[3]), "n"(kXStep), "n"(2 * kXStep), "n"(3 * kXStep)
      : "memory");
}

// Where the 16-byte chunks of row r of a tile of x stand in LDS: chunk c at c ^ this.  One LDS read of 16 bytes serves 16
// lanes at a time, rows 0-3 and 12-15 of one block of columns with rows 4-11 of the next one's (counted: with r & 7 those
// meet half of the banks twice, except where the lanes take neighbouring chunks of 128-byte rows), which then lie apart:
// 256-byte rows, blocks 4 chunks apart; 128-byte rows, blocks 2 apart.
__device__ inline int swizzle4(int r) { return (r & 3) | ((r & 8) != 0 ? 12 : 0); }
__device__ inline int swizzle2(int r) { return ((r >> 1) & 1) | ((r >> 1) & 4); }

// All loads of the wave but the last kLeft have arrived (those to LDS too).
template <int kLeft>
__device__ inline void wait_and_sync() {
  static_assert(kLeft < 64, "vmcnt has six bits");
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0x0070 | (kLeft & 15) | (kLeft >> 4) << 14);
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// A wave's lanes exchange data through LDS: what they wrote before is what they read behind this.  (No instruction: a wave's
// LDS accesses keep their order; the compiler has to keep it too.)
__device__ inline void wave_exchange() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront", "local");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront", "local");
}

// An offset past every buffer (they hold less than 2^30 bytes and a row's columns 2^21): loads give zeros.
constexpr int kOutside = 0x60000000;

// Four neighbouring outputs of row m.
__device__ inline void store_out(const LinearParams& p, int m, int n, f32x4 v) {
  uint16_t* out = p.out + m * p.out_stride;
  if (p.vector_out && n + 4 <= p.N) {
    if (p.bias != nullptr) {
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] += bf16_bits_to_f32(p.bias[n + e]);
    }
    *reinterpret_cast<uint2*>(out + n) = make_uint2(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]));
    return;
  }
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (n + e < p.N) out[n + e] = f32_to_bf16_bits(v[e] + (p.bias ? bf16_bits_to_f32(p.bias[n + e]) : 0.f));
}

// What a wave holds of one step of columns of the weight, and the scales of MX8 rows.
template <int MT, int NT>
struct Step {
  uint4 codes[NT][kStepTiles];
  uint32_t scale[NT];
  uint32_t xs[MT];  // lane 16 t + row: the four scale bytes of the row in tile t
};

// One workgroup per (NT * 8 / KS row tiles of the weight, MT tiles of 16 rows of x).  Its 8 waves form groups of KS that
// share NT row tiles; wave ks of a group takes steps ks, ks + KS, ... of 256 columns, and the group's sums are added
// through LDS, in the waves' order.
// Bound by HBM: the weight's 4.25 bits a value, read once for up to 32 rows of x, converted in registers (one instruction
// for two values) for bf16 matrix instructions; MX8 rows are converted too (exact products; the scaled matrix instruction
// would save 64 conversions per 2,048 weights of a wave, not time).  The loads of two steps are in flight.
// us per call with cold weights, bf16 / MX8 rows, beside a plain read of the same bytes: 28672 x 4096 for 1 row 15.4 / 14.9
// (read 12.3), for 32 19.0 / 18.5; 4096 x 14336 for 1 row 11.0 / 10.8 (read 6.6-8.7), for 32 16.8 / 14.2; 4096 x 4096 for 1 row
// 4.8 / 4.8 (read 3.5), for 32 6.7 / 6.1; bf16 weights in the library's GEMM: 28672 x 4096 for 32 rows 48.8, 4096 x 4096 13.8.
// The matrix instruction wants a different row of x in neighbouring lanes, which the L1 would serve 16 bytes a cycle:
// rows are loaded along their columns (64 bytes a cycle) and turned in a wave's own corner of LDS, its 16-byte chunks
// swizzled by the row so that neither side meets a bank twice (4096 x 4096 for 32 rows
// 10.6 -> 6.8 us).
template <bool kMx8, int MT, int NT, int KS>
__global__ __launch_bounds__(kWaves * 64, MT == 1 && NT == 1 ? 4 : 2) void mx4_rows_kernel(const LinearParams p) {
  constexpr int kLoads = kMx8 ? 2 : 4;  // of 1 KiB per tile of 16 rows x 128 columns
  constexpr int kRowBytes = kMx8 ? 128 : 256;  // of a row in a tile
  constexpr int kChunks = kRowBytes / 16;
  constexpr int kStage = MT * 16 * kRowBytes;
  constexpr int kPart = KS == 1 ? 0 : NT * MT * 64 * sizeof(f32x4);
  __shared__ __attribute__((aligned(16))) char smem[kWaves * (kStage > kPart ? kStage : kPart)];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = lane & 15, g = lane >> 4;
  const int ks = wave % KS;
  const int nt0 = (blockIdx.x * (kWaves / KS) + wave / KS) * NT, m0 = blockIdx.y * (16 * MT);
  const int ntiles = (p.N + 15) >> 4;
  f32x4 acc[NT][MT];
#pragma unroll
  for (int i = 0; i < NT; ++i)
#pragma unroll
    for (int j = 0; j < MT; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  const uint8_t* w[NT];
#pragma unroll
  for (int i = 0; i < NT; ++i) w[i] = p.w + static_cast<int64_t>(min(nt0 + i, ntiles - 1)) * p.tile_stride;
  const int valid = min(p.M - m0, 16 * MT);
  const int stride = static_cast<int>(p.x_stride) * (kMx8 ? 1 : 2), row_bytes = p.K * (kMx8 ? 1 : 2);
  const __amdgpu_buffer_rsrc_t xb = __builtin_amdgcn_make_buffer_rsrc(
      const_cast<char*>(static_cast<const char*>(p.x) + static_cast<int64_t>(m0) * stride), 0,
      (valid - 1) * stride + row_bytes, 0x00020000);
  const int lrow = lane / kChunks, lcol = (lane % kChunks) * 16;  // what this lane loads of a 1 KiB piece
  const int steps = (p.K + kStepCols - 1) / kStepCols;
  char* stage = smem + wave * kStage;

  auto load = [&](int h, Step<MT, NT>& st) {
    const int64_t unit = static_cast<int64_t>(h >> 1) * kMxUnitBytes;
#pragma unroll
    for (int i = 0; i < NT; ++i) {
#pragma unroll
      for (int t = 0; t < kStepTiles; ++t)
        st.codes[i][t] = load_nt(w[i] + unit + ((h & 1) * kStepTiles + t) * kMxTileBytes + lane * 16);
      st.scale[i] = reinterpret_cast<const uint32_t*>(w[i] + unit + 4 * kMxTileBytes)[lane];
    }
    if constexpr (kMx8) {
      const int b0 = h * (kStepCols / 32) + 4 * (lane >> 4), blocks = p.K >> 5;
#pragma unroll
      for (int j = 0; j < MT; ++j) {
        const uint8_t* s = p.xs + static_cast<int64_t>(m0 + min(16 * j + r, valid - 1)) * p.xs_stride + b0;
        uint32_t v = 0;
        if (lane < 16 * kStepTiles) {
          if (b0 + 4 <= blocks) {
            __builtin_memcpy(&v, s, 4);
          } else {
            for (int q = 0; q < 4; ++q)
              if (b0 + q < blocks) v |= static_cast<uint32_t>(s[q]) << (8 * q);
          }
        }
        st.xs[j] = v;
      }
    }
  };
  uint4 xr[MT][kLoads];  // the next tile of x, as loaded (16 bytes a lane, neighbouring lanes neighbouring bytes)
  auto load_x = [&](int tile) {
    const int col = tile * kRowBytes + lcol;
#pragma unroll
    for (int j = 0; j < MT; ++j)
#pragma unroll
      for (int i = 0; i < kLoads; ++i) {
        const int row = 16 * j + i * (64 / kChunks) + lrow;
        xr[j][i] = buffer_load16(xb, col < row_bytes && row < valid ? row * stride + col : kOutside);
      }
  };
  auto store_x = [&] {
#pragma unroll
    for (int j = 0; j < MT; ++j)
#pragma unroll
      for (int i = 0; i < kLoads; ++i) {
        const int row = i * (64 / kChunks) + lrow;
        *reinterpret_cast<uint4*>(stage + (16 * j + row) * kRowBytes + (lcol ^ ((kMx8 ? swizzle2(row) : swizzle4(row)) * 16))) = xr[j][i];
      }
  };
  auto compute = [&](int h, int t, const Step<MT, NT>& st) {
    const int byte = (h & 1) * kStepTiles + t;
    // lane (row, g) takes block g's 32 columns: step s of the matrix instruction, 8 of them
    float sx[MT];
    uint4 lo[MT], hi[MT];
    if constexpr (kMx8) {
#pragma unroll
      for (int j = 0; j < MT; ++j) {
        sx[j] = e8m0(__shfl(st.xs[j], 16 * t + r) >> (8 * g), 0);
        const char* at = stage + (16 * j + r) * kRowBytes;
        lo[j] = *reinterpret_cast<const uint4*>(at + ((32 * g) ^ (swizzle2(r) * 16)));
        hi[j] = *reinterpret_cast<const uint4*>(at + ((32 * g + 16) ^ (swizzle2(r) * 16)));
      }
    }
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      uint4 b[MT];
#pragma unroll
      for (int j = 0; j < MT; ++j) {
        if constexpr (kMx8)
          b[j] = s == 0   ? e4m3_to_bf16(lo[j].x, lo[j].y, sx[j])
                 : s == 1 ? e4m3_to_bf16(lo[j].z, lo[j].w, sx[j])
                 : s == 2 ? e4m3_to_bf16(hi[j].x, hi[j].y, sx[j])
                          : e4m3_to_bf16(hi[j].z, hi[j].w, sx[j]);
        else
          b[j] = *reinterpret_cast<const uint4*>(stage + (16 * j + r) * kRowBytes + ((64 * g + 16 * s) ^ (swizzle4(r) * 16)));
      }
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        const uint4 a = e2m1_to_bf16(word_of(st.codes[i][t], s), e8m0(st.scale[i], byte));
#pragma unroll
        for (int j = 0; j < MT; ++j) acc[i][j] = mfma_bf16(a, b[j], acc[i][j]);
      }
    }
  };

  // The codes of two steps ahead are in flight.  Three steps in turn, so that no loaded one is copied (a copy would wait).
  Step<MT, NT> s0, s1, s2;
  auto step = [&](int h, const Step<MT, NT>& now, Step<MT, NT>& then) {
    if (h + 2 * KS < steps) load(h + 2 * KS, then);
#pragma unroll
    for (int t = 0; t < kStepTiles; ++t) {
      wave_exchange();  // (the last tile has been read)
      store_x();
      wave_exchange();
      if (t + 1 < kStepTiles)
        load_x(h * kStepTiles + t + 1);
      else if (h + KS < steps)
        load_x((h + KS) * kStepTiles);
      compute(h, t, now);
    }
  };
  if (ks < steps) {
    load(ks, s0);
    load_x(ks * kStepTiles);
    if (ks + KS < steps) load(ks + KS, s1);
  }
  for (int h = ks; h < steps; h += 3 * KS) {
    step(h, s0, s2);
    if (h + KS < steps) step(h + KS, s1, s0);
    if (h + 2 * KS < steps) step(h + 2 * KS, s2, s1);
  }
  f32x4* part = reinterpret_cast<f32x4*>(smem);  // [wave][NT][MT][lane]
  if constexpr (KS > 1) {
    __syncthreads();
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
      for (int j = 0; j < MT; ++j) part[((wave * NT + i) * MT + j) * 64 + lane] = acc[i][j];
    __syncthreads();
  }
  // the KS waves of a group of columns take its NT x MT tiles in turn
#pragma unroll
  for (int q = 0; q < NT * MT; ++q) {
    if (q % KS != ks) continue;
    const int i = q / MT, j = q % MT;
    const int n = (nt0 + i) * 16 + 4 * g, m = m0 + 16 * j + r;
    f32x4 s = acc[i][j];
    if constexpr (KS > 1) {
      const f32x4* from = part + ((wave / KS) * KS * NT * MT + q) * 64 + lane;
      s = from[0];
#pragma unroll
      for (int v = 1; v < KS; ++v) s += from[v * NT * MT * 64];
    }
    if (m < p.M) store_out(p, m, n, s);
  }
}

// Many rows: one workgroup of WN x WM waves per (16 WN TN rows of the weight, 16 WM TM rows of x), each wave TN x TM
// tiles of 16 x 16.  Tiles of 128 columns go to LDS by direct loads, kBufs buffers in turn, one barrier a tile; two
// or three workgroups share a CU where there are that many, so that one's products cover the other's reads of LDS.
// MX8 rows: both operands and both scales go to the scaled matrix instruction as they are (a code is converted nowhere).
// Bound by the waits for the next tile: 4096 rows of 28672 x 4096 reach 2.47-2.57 PFLOP/s (375-389 us; bf16 weights in the
// library's GEMM 641 us), the matrix pipes 56 % busy; independent products in registers reach 3.83 PFLOP/s on this card, this
// loop without its loads 3.4.  With
// the tile staged through registers the same took 30-50 us more, with the outputs stored from registers 28.
// bf16 rows: the codes are converted in registers as they are used, by waves side by side over the weight (WM = 1), so that
// each is converted once and goes to its wave's registers only.  1000 rows of 6144 x 4096 take 44-47 us, 1.07-1.14 PFLOP/s, 4096 rows
// 151 us, 1.36 PFLOP/s (library, bf16 weights, 1000 rows: 52 us); bf16 products in registers reach 1.92 PFLOP/s.
template <bool kMx8, int WN, int WM, int TN, int TM, int kBufs>
__global__ __launch_bounds__(WN * WM * 64, 2) void mx4_tile_kernel(const LinearParams p, int mtiles, int grid) {
  constexpr int kThreads = WN * WM * 64, kBN = WN * TN, kBM = WM * TM;  // (in tiles of 16)
  constexpr int kRowBytes = kMx8 ? 128 : 256, kChunks = kRowBytes / 16;
  constexpr bool kOwnCodes = WM == 1;  // a wave's codes are no other's: to registers, the next tile's during the products
  constexpr int kXBytes = kBM * 16 * kRowBytes, kWBytes = kOwnCodes ? 0 : kBN * kMxTileBytes;
  constexpr int kBuf = kXBytes + kWBytes;
  constexpr int kXLoads = kBM * 16 * kChunks / kThreads, kWLoads = kOwnCodes ? TN : kBN * 64 / kThreads;
  constexpr int kLoads = kXLoads + kWLoads;  // of a tile
  static_assert(!kOwnCodes || 4 % (kBufs - 1) == 0, "tile t of a unit has its codes in place t % (kBufs - 1)");
  static_assert(kBufs == 2 || (kMx8 ? TN == 4 && TM == 2 : kOwnCodes && TM == 4), "the tiles of read_mx8 and read_bf16");
  constexpr int kOutRow = kBN * 32 + 16;  // bytes of an output row in LDS; the 16 spread the rows over the banks
  __shared__ __attribute__((aligned(16))) char smem[std::max(kBufs * kBuf, kBM * 16 * kOutRow)];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r = lane & 15, g = lane >> 4, wn = wave % WN, wm = wave / WN;
  // an XCD's workgroups in a row share four tiles of x and walk over the weight
  const int id = xcd_logical_index(blockIdx.x, grid);
  const int ntiles = (p.N + 15) >> 4, nblocks = (ntiles + kBN - 1) / kBN;
  const int group = id / (4 * nblocks), in_group = id % (4 * nblocks);
  const int rows_in_group = min(4, mtiles - 4 * group);
  const int mb = 4 * group + in_group % rows_in_group, nb = in_group / rows_in_group;
  const int m0 = mb * kBM * 16, nt0 = nb * kBN;

  const int valid = min(p.M - m0, kBM * 16), blocks = p.K >> 5;
  const int stride = static_cast<int>(p.x_stride) * (kMx8 ? 1 : 2), row_bytes = p.K * (kMx8 ? 1 : 2);
  const __amdgpu_buffer_rsrc_t xb = __builtin_amdgcn_make_buffer_rsrc(
      const_cast<char*>(static_cast<const char*>(p.x) + static_cast<int64_t>(m0) * stride), 0,
      (valid - 1) * stride + row_bytes, 0x00020000);
  const int wtiles = min(kBN, ntiles - nt0);
  const __amdgpu_buffer_rsrc_t wb = __builtin_amdgcn_make_buffer_rsrc(
      const_cast<uint8_t*>(p.w + static_cast<int64_t>(nt0) * p.tile_stride), 0, wtiles * p.tile_stride, 0x00020000);
  int wtile[TN], wload[kWLoads];  // starts of the wave's row tiles, and of those that it moves
#pragma unroll
  for (int i = 0; i < TN; ++i) wtile[i] = mx4_tile_start(wn * TN + i, wtiles, p.tile_stride);
#pragma unroll
  for (int j = 0; j < kWLoads; ++j)
    wload[j] = mx4_tile_start(kOwnCodes ? wn * TN + j : j * (kThreads / 64) + wave, wtiles, p.tile_stride);

  // what this lane moves: 16 bytes of rows xrow, xrow + kRowStep, ... of x, 16 of a lane's in every code tile.  LDS takes a
  // wave's bytes in lane order, so the lane picks the chunk that its place in the swizzled row holds.
  constexpr int kRowStep = kThreads / kChunks;
  static_assert(kRowStep % 16 == 0, "a lane's rows share their swizzle");
  const int xrow = tid / kChunks, xcol = ((tid % kChunks) ^ (kMx8 ? xrow & 7 : swizzle4(xrow))) * 16;
  int xoff[kXLoads];
#pragma unroll
  for (int j = 0; j < kXLoads; ++j)
    xoff[j] = xrow + j * kRowStep < valid ? (xrow + j * kRowStep) * stride + xcol : kOutside;
  uint4 codes[kBufs - 1][TN];  // of the next tiles
  auto load = [&](int kt, char* buf, int slot) {
    const bool in = xcol < row_bytes - kt * kRowBytes;
#pragma unroll
    for (int j = 0; j < kXLoads; ++j)
      buffer_to_lds16(xb, buf + wave * 1024 + j * kThreads * 16, in ? xoff[j] : kOutside, kt * kRowBytes);
    if constexpr (kOwnCodes) {
#pragma unroll
      for (int i = 0; i < TN; ++i)
        codes[slot][i] = buffer_load16(wb, lane * 16, wload[i] + mx4_codes_at(kt));
      return;
    }
#pragma unroll
    for (int j = 0; j < kWLoads; ++j)
      buffer_to_lds16(wb, buf + kXBytes + wave * 1024 + j * kThreads * 16, lane * 16, wload[j] + mx4_codes_at(kt));
  };

  f32x4 acc[TN][TM];
#pragma unroll
  for (int i = 0; i < TN; ++i)
#pragma unroll
    for (int j = 0; j < TM; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  // scales of this unit and the next, a byte a tile.  Of x lane (row, g) wants block g of every tile; it loads the four
  // blocks of tile g, whatever their alignment, and the four lanes of a row turn their bytes into each other's.
  uint32_t ws[TN], ws_next[TN], xs[TM], xs_next[TM];
  const uint8_t* const xs_base = p.xs + static_cast<int64_t>(m0) * p.xs_stride;
  int xs_row[TM];
  if constexpr (kMx8) {
#pragma unroll
    for (int j = 0; j < TM; ++j) xs_row[j] = min((wm * TM + j) * 16 + r, valid - 1) * static_cast<int>(p.xs_stride);
  }
  auto load_scales = [&](int u) {
#pragma unroll
    for (int i = 0; i < TN; ++i)
      ws_next[i] = __builtin_amdgcn_raw_buffer_load_b32(wb, lane * 4, wtile[i] + mx4_scales_at(u), 0);
    if constexpr (kMx8) {
      const int b0 = 16 * u + 4 * g;
      if (16 * u + 16 <= blocks) {
#pragma unroll
        for (int j = 0; j < TM; ++j) __builtin_memcpy(&xs_next[j], xs_base + xs_row[j] + b0, 4);
      } else {  // past the last block its scale: the products there are zero, or its NaN
#pragma unroll
        for (int j = 0; j < TM; ++j) {
          xs_next[j] = 0;
#pragma unroll
          for (int q = 0; q < 4; ++q) xs_next[j] |= static_cast<uint32_t>(xs_base[xs_row[j] + min(b0 + q, blocks - 1)]) << (8 * q);
        }
      }
    }
  };
  // (v_perm_b32: bytes 0-3 of the second operand, 4-7 of the first)
  const uint32_t turn16 = (g & 1) == 0 ? 0x06020400u : 0x03070105u, turn32 = (g & 2) == 0 ? 0x05040100u : 0x03020706u;
  auto next_unit = [&] {
#pragma unroll
    for (int i = 0; i < TN; ++i) ws[i] = ws_next[i];
    if constexpr (kMx8) {
#pragma unroll
      for (int j = 0; j < TM; ++j) {
        const uint32_t v = __builtin_amdgcn_perm(__shfl_xor(xs_next[j], 16), xs_next[j], turn16);
        xs[j] = __builtin_amdgcn_perm(__shfl_xor(v, 32), v, turn32);
      }
    }
  };

  const int tiles = (p.K + 127) >> 7;
  // tile kt: the fragments are read, then the loads of tile kt + kBufs - 1 start, which the products cover (past the last
  // tile they repeat it)
  char* now = smem;
  auto after = [&](char* buf, int n) {  // the buffer n further round
    char* q = buf + n * kBuf;
    return q < smem + kBufs * kBuf ? q : q - kBufs * kBuf;
  };
  auto step = [&](int k0, int t, bool rest) {
    const int kt = k0 + t;
    auto start_loads = [&] {
      __builtin_amdgcn_sched_barrier(0);
      if (t == 0) load_scales(min((kt >> 2) + 1, p.units - 1));
      load(min(kt + kBufs - 1, tiles - 1), after(now, kBufs - 1), t % (kBufs - 1));
      __builtin_amdgcn_sched_barrier(0);
    };
    const char* x = now + wm * TM * 16 * kRowBytes;
    const uint4* w = reinterpret_cast<const uint4*>(now + kXBytes + wn * TN * kMxTileBytes) + lane;
    uint4 c[TN];
    if constexpr (kOwnCodes) {
#pragma unroll
      for (int i = 0; i < TN; ++i) c[i] = codes[t % (kBufs - 1)][i];
    } else if constexpr (kBufs == 2) {
#pragma unroll
      for (int i = 0; i < TN; ++i) c[i] = w[i * 64];
    }
    if constexpr (kMx8) {
      // x: lane (row, g) takes columns 16 g .. and 64 + 16 g .. of a tile
      const char* row = x + r * kRowBytes;
      const char *at_lo = row + ((g ^ (r & 7)) * 16), *at_hi = row + (((g + 4) ^ (r & 7)) * 16);
      uint4 lo[TM], hi[TM];
      if constexpr (kBufs > 2) {
        read_mx8<16 * kRowBytes>(lds_address(w), lds_address(at_lo), lds_address(at_hi), c, lo, hi);
      } else {
#pragma unroll
        for (int j = 0; j < TM; ++j) {
          lo[j] = *reinterpret_cast<const uint4*>(at_lo + j * 16 * kRowBytes);
          hi[j] = *reinterpret_cast<const uint4*>(at_hi + j * 16 * kRowBytes);
        }
      }
      i32x8 b[TM];
#pragma unroll
      for (int j = 0; j < TM; ++j)
        b[j] = i32x8{(int)lo[j].x, (int)lo[j].y, (int)lo[j].z, (int)lo[j].w, (int)hi[j].x, (int)hi[j].y, (int)hi[j].z, (int)hi[j].w};
      start_loads();
#pragma unroll
      for (int i = 0; i < TN; ++i) {
        const i32x8 a = {(int)c[i].x, (int)c[i].y, (int)c[i].z, (int)c[i].w, 0, 0, 0, 0};
#pragma unroll
        for (int j = 0; j < TM; ++j)
          acc[i][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b[j], acc[i][j], 4, 0, 0, ws[i] >> (8 * t), 0, xs[j] >> (8 * t));
      }
    } else {
      uint4 b[4][TM];
      const char* at[4];
#pragma unroll
      for (int s = 0; s < 4; ++s) at[s] = x + r * kRowBytes + (((4 * g + s) ^ swizzle4(r)) * 16);
      if constexpr (kBufs > 2) {
        const uint32_t xa[4] = {lds_address(at[0]), lds_address(at[1]), lds_address(at[2]), lds_address(at[3])};
        read_bf16<16 * kRowBytes>(xa, b);
      } else {
#pragma unroll
        for (int s = 0; s < 4; ++s)
#pragma unroll
          for (int j = 0; j < TM; ++j) b[s][j] = *reinterpret_cast<const uint4*>(at[s] + j * 16 * kRowBytes);
      }
      start_loads();
#pragma unroll
      for (int s = 0; s < 4; ++s) {
#pragma unroll
        for (int i = 0; i < TN; ++i) {
          const uint4 a = e2m1_to_bf16(word_of(c[i], s), e8m0(ws[i], t));
#pragma unroll
          for (int j = 0; j < TM; ++j) acc[i][j] = mfma_bf16(a, b[s][j], acc[i][j]);
        }
      }
    }
    // the products come before the wait: nothing else orders them, and the compiler would move them behind it
#pragma unroll
    for (int i = 0; i < TN; ++i)
#pragma unroll
      for (int j = 0; j < TM; ++j) asm volatile("" : "+v"(acc[i][j]));
    __builtin_amdgcn_sched_barrier(0);
    // tile kt + 1 has arrived: all but the last kBufs - 2 steps' loads.  In the rest the compiler drops the codes that no
    // step reads any more, so that the steps issue fewer than kLoads: there all have arrived.
    if (kOwnCodes && rest)
      wait_and_sync<0>();
    else
      wait_and_sync<(kBufs - 2) * kLoads>();
    now = after(now, 1);
  };
  load_scales(0);
#pragma unroll
  for (int i = 0; i + 1 < kBufs; ++i) load(min(i, tiles - 1), smem + i * kBuf, i);
  wait_and_sync<0>();
  // (the four tiles of a unit without branches, so that the compiler can count the loads since the unit's scale words and
  // waits for those alone)
  const int full = tiles >> 2;
  for (int u = 0; u < full; ++u) {
    next_unit();
#pragma unroll
    for (int t = 0; t < 4; ++t) step(4 * u, t, false);
  }
  if (full < p.units) {
    next_unit();
#pragma unroll
    for (int t = 0; t < 3; ++t)
      if (t < (tiles & 3)) step(4 * full, t, true);
  }
  if constexpr (kBufs > 2) wait_and_sync<0>();  // (the loads past the last tile still write the buffers)
  // The outputs go through LDS into whole rows: a lane's four stand 32 bytes wide in 16 rows, which HBM takes at 2 TB/s
  // (4096 rows of 28672 x 4096: 394 us).
#pragma unroll
  for (int i = 0; i < TN; ++i) {
    const int col = (wn * TN + i) * 16 + 4 * g, n = nt0 * 16 + col;
    float bias[4] = {0.f, 0.f, 0.f, 0.f};
    if (p.bias != nullptr) {
#pragma unroll
      for (int e = 0; e < 4; ++e) bias[e] = n + e < p.N ? bf16_bits_to_f32(p.bias[n + e]) : 0.f;
    }
#pragma unroll
    for (int j = 0; j < TM; ++j) {
      const f32x4 v = acc[i][j];
      *reinterpret_cast<uint2*>(smem + ((wm * TM + j) * 16 + r) * kOutRow + col * 2) =
          make_uint2(pack_bf16x2(v[0] + bias[0], v[1] + bias[1]), pack_bf16x2(v[2] + bias[2], v[3] + bias[3]));
    }
  }
  __syncthreads();
  constexpr int kPieces = kBN * 2;  // of 16 bytes in a row
#pragma unroll 4
  for (int q = tid; q < kBM * 16 * kPieces; q += kThreads) {
    const int row = q / kPieces, n = nt0 * 16 + (q % kPieces) * 8;
    if (row >= valid || n >= p.N) continue;
    const uint4 v = *reinterpret_cast<const uint4*>(smem + row * kOutRow + (q % kPieces) * 16);
    uint16_t* out = p.out + static_cast<int64_t>(m0 + row) * p.out_stride + n;
    if (p.vector_out && n + 8 <= p.N) {
      *reinterpret_cast<uint4*>(out) = v;
    } else {
      const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (n + e < p.N) out[e] = static_cast<uint16_t>(u[e >> 1] >> (16 * (e & 1)));
    }
  }
}

template <bool kMx8, int MT, int NT, int KS>
void launch_rows(const LinearParams& p, hipStream_t s) {
  constexpr int kTiles = NT * kWaves / KS;  // row tiles of a workgroup
  const dim3 grid(static_cast<unsigned>((p.N + 16 * kTiles - 1) / (16 * kTiles)),
                  static_cast<unsigned>((p.M + 16 * MT - 1) / (16 * MT)));
  mx4_rows_kernel<kMx8, MT, NT, KS><<<grid, kWaves * 64, 0, s>>>(p);
}

// One round of workgroups, one per CU: `per` row tiles of the weight each.  More workgroups read x more often and wait
// for each other's start and end (4096 x 4096 for 64 rows, us: 10.7 with 512, 7.9 with 256); fewer leave CUs idle (128:
// 12.0).  For four tiles a workgroup the waves split the columns rather than the rows (14336 x 4096 for 32 rows: 12.3
// against 14.1 with two tiles and half the columns each).
template <bool kMx8, int MT>
void launch_mt(const LinearParams& p, hipStream_t s) {
  const int64_t cus = std::max(1, device_cu_count());
  const int64_t tiles = static_cast<int64_t>((p.N + 15) / 16) * ((p.M + 16 * MT - 1) / (16 * MT));
  const int64_t per = (tiles + cus - 1) / cus;
  if (per <= 1)
    launch_rows<kMx8, MT, 1, 8>(p, s);
  else if (per <= 2)
    launch_rows<kMx8, MT, 2, 8>(p, s);
  else if (per <= 4)
    launch_rows<kMx8, MT, 4, 8>(p, s);
  else if (per <= 8)
    launch_rows<kMx8, MT, 4, 4>(p, s);
  else if (per <= 16)
    launch_rows<kMx8, MT, 4, 2>(p, s);
  else
    launch_rows<kMx8, MT, 4, 1>(p, s);
}

template <bool kMx8, int WN, int WM, int TN, int TM, int kBufs>
void launch_tile(const LinearParams& p, hipStream_t s) {
  const int nblocks = (p.N + 16 * WN * TN - 1) / (16 * WN * TN), mtiles = (p.M + 16 * WM * TM - 1) / (16 * WM * TM);
  const int grid = nblocks * mtiles;
  mx4_tile_kernel<kMx8, WN, WM, TN, TM, kBufs><<<grid, WN * WM * 64, 0, s>>>(p, mtiles, grid);
}

// The tile kernel where the row kernel would give each CU more than 8 tiles of 16 weight rows x 32 rows of x, for MX8 rows
// more than 4: a round of tiles takes as long whether it fills its CUs or not (us, row kernel against tiles.  bf16 rows:
// 4096 x 14336 for 256 rows, 8 tiles a CU, 44.8 against 68.6; 6968 x 2592 for 143, 8.5, 21.1 against 15.4; 14336 x 4096 for 96,
// 10.5, 27.0 against 23.2; 6144 x 4096 for 256, 12, 25.1 against 22.9; 28672 x 4096 for 64, 14, 29.0 against 24.2.  MX8 rows:
// 4096 x 14336 for 128 rows, 4, 25.3 against 46; 2387 x 11744 for 201, 4.1, 48 against 37; 6144 x 4096 for 128, 6, 15.5
// against 16.7; 28672 x 4096 for 32, 7, 19.3 against 18.3; 14336 x 4096 for 96, 10.5, 27.4 against 16.1).  At any width the
// row kernel, which HBM bounds, for up to 32 bf16 rows (128256 x 4096: 62 against 97) and up to 16 MX8 rows, whose products it
// takes exactly.
// Large tiles where 128 x 64 ones would be more than three a CU (us, MX8 rows: 28672 x 4096 for 4096 rows 375 with
// 256 x 128, 459 with 128 x 128; 6144 x 4096 for 1000 rows, three a CU, 37.7 against 32.6 with 128 x 64.  bf16 rows: 28672 x
// 4096 for 4096 rows 690 with 256 x 64, 722 with 128 x 128; for 256 rows, 3.5 a CU, 52 against 61 with 128 x 64; 4096 x 14336 for
// 1000 rows, two a CU, 110 against 101).
// Small MX8 tiles take four buffers while that leaves a CU its two workgroups, as few of them wait for memory most of the
// time, and three for the third (us, two / three / four buffers: 4096 x 14336 for 256 rows, one for two CUs, 84 / 53 / 46;
// for 1000 rows, two a CU, 85 / 71 / 67; 6144 x 4096 for 1000, three a CU, 31.9 / 32.6 / 36.3).  bf16: three (two / three /
// five: 4096 x 14336 for 256 rows 93 / 68 / 73; for 1000, 101 / 101 / 110), large tiles two (28672 x 4096 for 4096 rows, two /
// three, 690 / 709).
template <bool kMx8>
int32_t launch(const LinearParams& p, hipStream_t s, int kernel) {
  const int64_t cus = std::max(1, device_cu_count());
  const int64_t work = static_cast<int64_t>((p.N + 15) / 16) * ((p.M + 31) / 32);
  if (kernel == LKV_MX4_TILES || (kernel == LKV_MX4_AUTO && p.M > (kMx8 ? 16 : 32) && work > (kMx8 ? 4 : 8) * cus)) {
    const int64_t small = static_cast<int64_t>((p.N + 127) / 128) * ((p.M + 63) / 64);  // tiles of 128 x 64
    if constexpr (kMx8) {
      if (small <= 2 * cus)
        launch_tile<true, 2, 2, 4, 2, 4>(p, s);
      else if (small <= 3 * cus)
        launch_tile<true, 2, 2, 4, 2, 3>(p, s);
      else
        launch_tile<true, 2, 2, 8, 4, 2>(p, s);
    } else {
      if (small <= 3 * cus)
        launch_tile<false, 4, 1, 2, 4, 3>(p, s);
      else
        launch_tile<false, 4, 1, 4, 4, 2>(p, s);
    }
  } else if (p.M <= 16) {
    launch_mt<kMx8, 1>(p, s);
  } else {
    launch_mt<kMx8, 2>(p, s);
  }
  return check_launch("lkv_mx4_linear");
}

// ---- packing (off the path) ----

// Lane l of tile t of a unit: its 16 code bytes and its scale byte.  Rows and columns past the matrix: zeros.
struct PackItem {
  int64_t at;  // of the unit's bytes
  int t, lane, n, k;
};

__device__ inline bool pack_item(int64_t id, int32_t units, int32_t N, int32_t K, PackItem& it) {
  it.lane = id & 63;
  it.t = (id >> 6) & 3;
  const int64_t tile = (id >> 8) / units;
  const int u = static_cast<int>((id >> 8) % units);
  it.at = tile * mx4_tile_stride(units) + u * kMxUnitBytes;
  it.n = static_cast<int>(tile) * 16 + (it.lane & 15);
  it.k = u * kMxUnitCols + it.t * 128 + 32 * (it.lane >> 4);
  return it.n < N && it.k < K;
}

__device__ inline void pack_store(uint8_t* out, const PackItem& it, uint4 codes, uint8_t scale) {
  uint8_t* unit = out + it.at;
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
    const uint8_t* unit = w + it.at;
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
  LKV_REQUIRE((n) > 0 && (n) <= (1 << 24) && (k) > 0 && (k) <= (1 << 20) && (k) % 32 == 0,                       \
              "an MX4 weight has 1 to 2^24 rows and a positive multiple of 32 columns up to 2^20, got %d x %d", n, k)

extern "C" int64_t lkv_mx4_weight_bytes(int32_t n, int32_t k) {
  if (n <= 0 || n > (1 << 24) || k <= 0 || k > (1 << 20)) return 0;
  return static_cast<int64_t>((n + 15) / 16) * lkv::mx4_tile_stride(lkv::mx4_units(k));
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
      static_cast<uint8_t*>(weight), n, k, mx4_units(k), items);
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
                                                                      mx4_units(k), items);
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
                                                                    mx4_units(k), items);
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
  LKV_REQUIRE(a->kernel >= LKV_MX4_AUTO && a->kernel <= LKV_MX4_TILES, "kernel must be one of LKV_MX4_*, got %d", a->kernel);
  const bool mx8 = a->x_format == LKV_X_MX8;
  LKV_REQUIRE(a->rows >= 0 && a->rows <= (1 << 20), "rows must be in [0, 2^20], got %d", a->rows);
  LKV_REQUIRE_MX4_SHAPE(a->out_features, a->in_features);
  LKV_REQUIRE(a->x != nullptr && a->weight != nullptr && a->out != nullptr, "null x/weight/out");
  LKV_REQUIRE(mx8 == (a->x_scales != nullptr), "x_scales belong to MX8 rows, and they need them");
  LKV_REQUIRE(((bits(a->x) | bits(a->weight)) & 15) == 0 && ((bits(a->out) | bits(a->bias)) & 1) == 0,
              "x and weight must be 16-byte aligned");
  if (a->rows > 1) {  // (one row has no stride)
    LKV_REQUIRE(a->x_stride % (mx8 ? 16 : 8) == 0, "x rows must be 16-byte aligned");
    LKV_REQUIRE(a->x_stride >= 0 && a->x_stride <= (1 << 21), "x_stride must be at most 2^21 elements");
    LKV_REQUIRE(!mx8 || (a->x_scale_stride >= 0 && a->x_scale_stride <= (1 << 21)), "x_scale_stride must be at most 2^21 bytes");
    LKV_REQUIRE(a->out_stride >= a->out_features, "out rows must not overlap");
  }
  if (a->rows == 0) return LKV_OK;
  LinearParams p;
  p.w = static_cast<const uint8_t*>(a->weight);
  p.x = a->x;
  p.x_stride = a->rows > 1 ? a->x_stride : 0;
  p.xs = static_cast<const uint8_t*>(a->x_scales);
  p.xs_stride = a->rows > 1 ? a->x_scale_stride : 0;
  p.bias = static_cast<const uint16_t*>(a->bias);
  p.out = static_cast<uint16_t*>(a->out);
  p.out_stride = a->rows > 1 ? a->out_stride : 0;
  p.M = a->rows;
  p.N = a->out_features;
  p.K = a->in_features;
  p.units = mx4_units(a->in_features);
  p.tile_stride = mx4_tile_stride(p.units);
  p.vector_out = (bits(a->out) & 15) == 0 && p.out_stride % 8 == 0;
  return mx8 ? launch<true>(p, as_stream(stream), a->kernel) : launch<false>(p, as_stream(stream), a->kernel);
}
