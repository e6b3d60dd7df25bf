// Beam search's selection: the `count` best of a prompt's beams x vocab candidates score + (logit - lse(beam's logits)).
//
// Inside one beam the order of the totals is the order of the logits, so one pass over the logits does all of the reading:
//   slice kernel: a workgroup holds a slice of one beam's row in registers (8 or 32 values a thread), takes its maximum,
//     the sum of its exponentials and its `count` greatest logits;
//   choose kernel: a workgroup a prompt joins the slices' sums in 64 bits and chooses among the slices' candidates.
// Choosing the n greatest of many values needs no sort: the n-th greatest of the threads' own maxima is a floor that at
// least n values reach and few others do; those go to LDS and each counts the ones before it.  Where too many values reach
// the floor for LDS (equal logits), n rounds take the next one each; both give the same set.
// 16 prompts of 8 beams of 128256 bf16 logits, 16 of each: slices 12.0 us (2.7 TB/s; 13.0 on the mean; the loads and the maximum
// alone 5.9, with the exponentials 8.2, so that a third is the choice and its barriers), choosing 6.9-7.6; one prompt of 4 beams of
// 32000 3.8-4.5 and 3.2-5.0, which are two dependent launches.
#include "common.h"
#include "runtime.h"

namespace lkv {
namespace {

constexpr int kBeamThreads = 256;
constexpr int kBeamCap = 1024;  // candidates that LDS takes
constexpr int kNarrowSlice = 2048, kWideSlice = 8192;
constexpr float kNegInf = -__builtin_inff();

struct SliceSum {
  double s;  // sum of exp(x - m)
  float m;
  int32_t pad;
};

struct BeamParams {
  const void* logits;
  int64_t sb, sk;
  const float* scores;
  int64_t scores_sb;
  float* out_scores;
  int32_t* out_beams;
  int32_t* out_tokens;
  SliceSum* sums;   // [B * K, slices]
  float* val;       // [B * K, slices, count]: logits
  int32_t* idx;     // tokens, -1: none
  int32_t beams, vocab, count, slices;
  float per_tile;   // beams in one tile of the choose kernel: 1 over a beam's tiles
};

// Monotone in x for every x but NaN; above 0.
__device__ inline uint32_t order_bits(float x) {
  const uint32_t u = __float_as_uint(x + 0.f);  // (-0 and +0 are equal)
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

__device__ inline float from_order(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }

template <int kCtrl>
__device__ inline float dpp_move(float x) {
  return __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(x), kCtrl, 0xf, 0xf, true));
}

// A floor that at least n (<= 64) of the values reach of which each of the kThreads threads gives the greatest: the n-th
// greatest of the maxima of 64 groups of neighbours, found by counting for each how many stand before it (a wave counts a
// part of them).  A group's number takes the place of its maximum's lowest six bits, so that one comparison decides; the
// floor is the n-th with those bits clear, at or below it.  64 groups are the fewest that do, and their counting the least
// (256 groups of four made the choice below 6.5 us where it takes 4.8, for one prompt of 4 beams).
template <int kThreads>
struct FloorShared {
  uint32_t top[64];
  uint32_t before[64];
  float result;
};

template <int kThreads>
__device__ inline float nth_floor(float x, int n, FloorShared<kThreads>& sm) {
  constexpr int kGroup = kThreads / 64, kWaves = kThreads / 64, kPart = 64 / kWaves;
  static_assert(kGroup == 4 || kGroup == 16, "groups are quads or rows of 16 lanes");
  const int t = threadIdx.x, i = t & 63, part = t >> 6;
  x = fmaxf(x, dpp_move<0xb1>(x));
  x = fmaxf(x, dpp_move<0x4e>(x));
  if (kGroup == 16) {
    x = fmaxf(x, dpp_move<0x141>(x));  // (the row's halves mirrored, then the row)
    x = fmaxf(x, dpp_move<0x140>(x));
  }
  if (t % kGroup == 0) sm.top[t / kGroup] = (order_bits(x) & ~63u) | static_cast<uint32_t>(t / kGroup);
  if (part == 0) sm.before[i] = 0;
  __syncthreads();
  const uint32_t mine = sm.top[i];
  uint32_t before = 0;
#pragma unroll
  for (int j = part * kPart; j < (part + 1) * kPart; j += 4) {
    const uint4 k = *reinterpret_cast<const uint4*>(&sm.top[j]);
    before += k.x > mine;
    before += k.y > mine;
    before += k.z > mine;
    before += k.w > mine;
  }
  atomicAdd(&sm.before[i], before);
  __syncthreads();
  if (part == 0 && sm.before[i] == static_cast<uint32_t>(n - 1))
    sm.result = from_order(max(mine & ~63u, 0x007fffffu));  // (-inf's place: those below are NaN)
  __syncthreads();
  return sm.result;
}

// Takes n places of a list in LDS.  (The 0 from the asm keeps the counter's address a vector register: seeing one address for
// the wave the compiler adds the lanes' shares up one lane after the other first; the slices of 128 rows took 12.0 us so,
// 11.4 this way.)
__device__ inline uint32_t take_places(uint32_t* counter, uint32_t n) {
  uint32_t zero;
  asm("v_mov_b32 %0, 0" : "=v"(zero));
  return atomicAdd(counter + zero, n);
}

// Sixteen bytes of a row, eight bf16 or four fp32 values from element e0 >= 0 on, where the row ends among or before them:
// elements from V on are not read and are -inf.
template <bool kF32>
__device__ inline uint4 last_piece(const void* row, int e0, int V) {
  uint32_t u[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if constexpr (kF32) {
      const int e = e0 + j;
      u[j] = e < V ? static_cast<const uint32_t*>(row)[e] : 0xff800000u;
    } else {
      const int e = e0 + 2 * j;
      const uint32_t lo = e < V ? static_cast<const uint16_t*>(row)[e] : 0xff80u;
      const uint32_t hi = e + 1 < V ? static_cast<const uint16_t*>(row)[e + 1] : 0xff80u;
      u[j] = lo | hi << 16;
    }
  }
  return make_uint4(u[0], u[1], u[2], u[3]);
}

// Sixteen bytes at the alignment of a row's values (the card loads dwords from any address).
template <bool kF32>
__device__ inline uint4 load_piece(const void* row, int e) {
  uint4 w;
  if constexpr (kF32)
    __builtin_memcpy(&w, static_cast<const float*>(row) + e, 16);
  else
    __builtin_memcpy(&w, static_cast<const uint16_t*>(row) + e, 16);
  return w;
}

template <bool kF32>
__device__ inline float value_of(const uint4& w, int j) {
  const uint32_t u[4] = {w.x, w.y, w.z, w.w};
  return kF32 ? __uint_as_float(u[j & 3]) : j & 1 ? bf16_hi(u[j >> 1]) : bf16_lo(u[j >> 1]);
}

template <bool kF32, int kChunks>
__global__ __launch_bounds__(kBeamThreads) void beam_slice_kernel(const BeamParams p) {
  constexpr int kVec = kF32 ? 4 : 8;
  __shared__ __align__(16) FloorShared<kBeamThreads> sm_floor;
  __shared__ uint64_t sm_cand[kBeamCap];
  __shared__ double sm_sum[4];
  __shared__ float sm_max[4];
  __shared__ uint32_t sm_n;
  __shared__ uint64_t sm_best[4];
  const int t = threadIdx.x, wave = t >> 6, lane = t & 63;
  const int slice = blockIdx.x, row_id = blockIdx.y, V = p.vocab, n = p.count;
  const int64_t off = (row_id / p.beams) * p.sb + (row_id % p.beams) * p.sk;
  const void* row = kF32 ? static_cast<const void*>(static_cast<const float*>(p.logits) + off)
                         : static_cast<const void*>(static_cast<const uint16_t*>(p.logits) + off);
  // Pieces are counted from the row's first value, whatever its address: which values a thread adds in fp32, and so every bit of
  // a row's sum, then goes by the row's values alone, and equal beams tie exactly.  (With pieces at multiples of 16 bytes the
  // logarithms of equal rows at different alignments differed by 1e-8, which put a later beam first.)
  const int e0 = (slice * kChunks * kBeamThreads + t) * kVec;  // this thread's first element
  constexpr int kStep = kBeamThreads * kVec;
  // Every thread's loads are issued before the first is waited for: pieces that are not the row's read one that is, and the
  // row's end is put right after that (with a branch at each load the loads followed one another, and 128 rows of 128256
  // took 1 us of 15 longer).
  const int tail = V / kVec * kVec - kVec;  // the row's last whole piece
  uint4 raw[kChunks];
  if (tail >= 0) {
#pragma unroll
    for (int c = 0; c < kChunks; ++c) raw[c] = load_piece<kF32>(row, min(e0 + c * kStep, tail));
  }
  if ((slice + 1) * kChunks * kStep > V) {
#pragma unroll
    for (int c = 0; c < kChunks; ++c)
      if (e0 + c * kStep > tail) raw[c] = last_piece<kF32>(row, e0 + c * kStep, V);
  }
  if (t == 0) sm_n = 0;
  float best = kNegInf, top[kChunks];  // (NaN where one is: its row then has no candidate, whatever the slices hold)
#pragma unroll
  for (int c = 0; c < kChunks; ++c) {
    top[c] = kNegInf;
#pragma unroll
    for (int j = 0; j < kVec; j += 2) top[c] = fmax3_nan(top[c], value_of<kF32>(raw[c], j), value_of<kF32>(raw[c], j + 1));
    best = fmax_nan(best, top[c]);
  }
  float m = best;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) m = fmax_nan(m, __shfl_xor(m, o));
  if (lane == 0) sm_max[wave] = m;
  const float floor = nth_floor(best, n, sm_floor);  // (its barriers publish sm_max and sm_n)
  m = fmax_nan(fmax_nan(sm_max[0], sm_max[1]), fmax_nan(sm_max[2], sm_max[3]));
  const int64_t out = (static_cast<int64_t>(row_id) * p.slices + slice);
  float* val = p.val + out * n;
  int32_t* idx = p.idx + out * n;
  if (m != m) {
    if (t == 0) p.sums[out] = SliceSum{__builtin_nan(""), kNegInf, 0};
    for (int r = t; r < n; r += kBeamThreads) idx[r] = -1;
    return;
  }
  // the values that reach the floor, as (order, lowest index first).  Few do: a thread looks into the pieces whose maximum
  // does, one after the other, and takes their values out by selects (a test of every value in every wave was 3 us of 14)
  auto key = [&](float v, int e) {
    return (static_cast<uint64_t>(order_bits(v)) << 32) | static_cast<uint32_t>(~static_cast<uint32_t>(e));
  };
  const float cut = fmaxf(floor, -3.402823466e38f);
  uint32_t pieces = 0;
#pragma unroll
  for (int c = 0; c < kChunks; ++c) pieces |= top[c] >= cut ? 1u << c : 0u;
  while (pieces != 0) {
    const int c = __builtin_ctz(pieces);
    pieces &= pieces - 1;
    uint32_t x = raw[0].x, y = raw[0].y, z = raw[0].z, o = raw[0].w;
#pragma unroll
    for (int k = 1; k < kChunks; ++k) {
      x = c == k ? raw[k].x : x;
      y = c == k ? raw[k].y : y;
      z = c == k ? raw[k].z : z;
      o = c == k ? raw[k].w : o;
    }
    const uint4 w = make_uint4(x, y, z, o);
    uint32_t hits = 0;
#pragma unroll
    for (int j = 0; j < kVec; ++j) hits |= value_of<kF32>(w, j) >= cut ? 1u << j : 0u;
    uint32_t at = take_places(&sm_n, static_cast<uint32_t>(__builtin_popcount(hits)));
    while (hits != 0) {
      const int j = __builtin_ctz(hits);
      hits &= hits - 1;
      const int word = kF32 ? j : j >> 1;
      const uint32_t u = word & 2 ? (word & 1 ? o : z) : (word & 1 ? y : x);
      const float v = kF32 ? __uint_as_float(u) : j & 1 ? bf16_hi(u) : bf16_lo(u);
      if (at < kBeamCap) sm_cand[at] = key(v, e0 + c * kStep + j);
      ++at;
    }
  }
  const float ref = m == kNegInf ? 0.f : m;  // (x - ref is 0 for the greatest, whose term is then exactly 1)
  float part = 0.f;
#pragma unroll
  for (int c = 0; c < kChunks; ++c)
#pragma unroll
    for (int j = 0; j < kVec; ++j) part += fast_exp2((value_of<kF32>(raw[c], j) - ref) * kLog2e);  // (a +inf makes it NaN)
  double sum = part;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o);
  if (lane == 0) sm_sum[wave] = sum;
  __syncthreads();
  if (t == 0) p.sums[out] = SliceSum{(sm_sum[0] + sm_sum[1]) + (sm_sum[2] + sm_sum[3]), m, 0};
  auto put = [&](int r, uint64_t c) {
    val[r] = from_order(static_cast<uint32_t>(c >> 32));
    idx[r] = static_cast<int32_t>(~static_cast<uint32_t>(c));
  };
  const int found = static_cast<int>(sm_n);
  for (int r = min(found, n) + t; r < n; r += kBeamThreads) idx[r] = -1;
  if (found <= kBeamCap) {
    for (int i = t; i < found; i += kBeamThreads) {
      const uint64_t mine = sm_cand[i];
      int before = 0;
#pragma unroll 8
      for (int k = 0; k < found; ++k) before += sm_cand[k] > mine;
      if (before < n) put(before, mine);
    }
    return;
  }
  uint64_t last = ~uint64_t{0};
  for (int r = 0; r < n; ++r) {  // the next one below the last, n times (more than n reach the floor)
    uint64_t next = 0;
#pragma unroll
    for (int c = 0; c < kChunks; ++c)
#pragma unroll
      for (int j = 0; j < kVec; ++j) {
        const float x = value_of<kF32>(raw[c], j);
        if (!(x > kNegInf)) continue;
        const uint64_t k = key(x, e0 + c * kStep + j);
        if (k < last && k > next) next = k;
      }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) next = max(next, static_cast<uint64_t>(__shfl_xor(static_cast<unsigned long long>(next), o)));
    if (lane == 0) sm_best[wave] = next;
    __syncthreads();
    next = max(max(sm_best[0], sm_best[1]), max(sm_best[2], sm_best[3]));
    if (t == 0) put(r, next);
    last = next;
    __syncthreads();
  }
}

// A candidate's total and what decides between equal ones: lowest beam, then greatest logit (its own total is the greater one
// before rounding), then lowest token.
struct Candidate {
  double total;
  uint64_t tie;  // 0: none
};

__device__ inline Candidate make_candidate(double total, int beam, float logit, int token) {
  return Candidate{total, (static_cast<uint64_t>(LKV_BEAM_MAX_BEAMS - 1 - beam) << 52) | (static_cast<uint64_t>(order_bits(logit)) << 20) |
                              static_cast<uint64_t>(0xfffff - token)};
}

__device__ inline bool ahead(const Candidate& a, const Candidate& b) {
  return a.total > b.total || (a.total == b.total && a.tie > b.tie);
}

// Candidates of the slices, 64 of one beam at a time ("tile"), tiles dealt to the waves; a wave keeps its first kHeld.
constexpr int kChooseThreads = 1024, kChooseWaves = kChooseThreads / 64, kHeld = 4;

__global__ __launch_bounds__(kChooseThreads) void beam_choose_kernel(const BeamParams p) {
  __shared__ __align__(16) FloorShared<kChooseThreads> sm_floor;
  __shared__ double sm_lse[LKV_BEAM_MAX_BEAMS], sm_score[LKV_BEAM_MAX_BEAMS], sm_total[kBeamCap], sm_wtotal[kChooseWaves];
  __shared__ uint64_t sm_tie[kBeamCap], sm_wtie[kChooseWaves];
  __shared__ uint32_t sm_n;
  const int t = threadIdx.x, lane = t & 63, b = blockIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const int K = p.beams, n = p.count, S = p.slices, per = S * n;
  const int tiles = (per + 63) / 64, all = K * tiles;
  const int64_t base = static_cast<int64_t>(b) * K * per;
  if (t == 0) sm_n = 0;
  // (there are at most 64 * 513 tiles, so that the product is closer to the quotient than that is to the next integer; an
  // integer division for every tile in every pass was 1 us of the kernel)
  auto beam_of = [&](int tile) { return static_cast<int>((static_cast<float>(tile) + 0.5f) * p.per_tile); };
  // the held tiles' tokens and logits are on their way while the sums are joined
  int token[kHeld];
  float logit[kHeld];
  auto fetch = [&](int tile, int& tk, float& x) {
    const int k = beam_of(tile), i = (tile - k * tiles) * 64 + lane;
    tk = -1;
    x = 0.f;
    if (i < per) {
      tk = p.idx[base + k * per + i];
      x = p.val[base + k * per + i];
    }
  };
#pragma unroll
  for (int h = 0; h < kHeld; ++h) {
    token[h] = -1;
    if (wave + h * kChooseWaves < all) fetch(wave + h * kChooseWaves, token[h], logit[h]);
  }
  for (int k = wave; k < K; k += kChooseWaves) {
    const SliceSum* ss = p.sums + (static_cast<int64_t>(b) * K + k) * S;
    float m = kNegInf;
    double s = 0;
    for (int i = lane; i < S; i += 64) {
      const SliceSum v = ss[i];  // (an empty slice's sum is 0, or NaN)
      const float to = fmaxf(m, v.m);
      if (m != to && m != kNegInf) s *= exp(static_cast<double>(m) - static_cast<double>(to));
      s += v.m == to || v.m == kNegInf ? v.s : v.s * exp(static_cast<double>(v.m) - static_cast<double>(to));
      m = to;
    }
    float top = m;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
    if (m != top && m != kNegInf) s *= exp(static_cast<double>(m) - static_cast<double>(top));
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o);
    if (lane == 0) {
      sm_lse[k] = static_cast<double>(top) + log(s);  // (-inf or NaN for a row without a candidate)
      sm_score[k] = p.scores[b * p.scores_sb + k];
    }
  }
  __syncthreads();
  auto candidate = [&](int tile, int tk, float x) {
    const int k = beam_of(tile);
    const double total = sm_score[k] + (static_cast<double>(x) - sm_lse[k]);
    return tk >= 0 && fabs(total) < __builtin_inf() ? make_candidate(total, k, x, tk) : Candidate{0, 0};
  };
  // f(candidate) for this lane's candidates of every tile
  auto each = [&](auto&& f) {
#pragma unroll
    for (int h = 0; h < kHeld; ++h)
      if (wave + h * kChooseWaves < all) f(candidate(wave + h * kChooseWaves, token[h], logit[h]));
    for (int tile = wave + kHeld * kChooseWaves; tile < all; tile += kChooseWaves) {
      int tk;
      float x;
      fetch(tile, tk, x);
      f(candidate(tile, tk, x));
    }
  };
  float top = kNegInf;  // (totals rounded down: a floor of them is one of the totals)
  each([&](const Candidate& c) {
    if (c.tie != 0) top = fmaxf(top, __double2float_rd(c.total));
  });
  const float floor = nth_floor(top, n, sm_floor);
  each([&](const Candidate& c) {
    if (c.tie != 0 && __double2float_rd(c.total) >= floor) {
      const uint32_t at = take_places(&sm_n, 1);
      if (at < kBeamCap) {
        sm_total[at] = c.total;
        sm_tie[at] = c.tie;
      }
    }
  });
  __syncthreads();
  const int found = static_cast<int>(sm_n);
  auto put = [&](int r, const Candidate& c) {
    const int64_t o = static_cast<int64_t>(b) * n + r;
    p.out_scores[o] = c.tie == 0 ? kNegInf : static_cast<float>(c.total);
    p.out_beams[o] = c.tie == 0 ? -1 : LKV_BEAM_MAX_BEAMS - 1 - static_cast<int>(c.tie >> 52);
    p.out_tokens[o] = c.tie == 0 ? -1 : 0xfffff - static_cast<int>(c.tie & 0xfffff);
  };
  for (int r = min(found, n) + t; r < n; r += kChooseThreads) put(r, Candidate{0, 0});
  if (found <= kBeamCap) {
    if (t < found) {
      const Candidate mine{sm_total[t], sm_tie[t]};
      int before = 0;
#pragma unroll 4
      for (int k = 0; k < found; ++k) before += ahead(Candidate{sm_total[k], sm_tie[k]}, mine);
      if (before < n) put(before, mine);
    }
    return;
  }
  Candidate last{0, 0};
  for (int r = 0; r < n; ++r) {  // the next one behind the last, n times
    Candidate best{0, 0};
    auto take = [&](const Candidate& c) {
      if (c.tie != 0 && (best.tie == 0 || ahead(c, best))) best = c;
    };
    each([&](const Candidate& c) {
      if (r == 0 || ahead(last, c)) take(c);
    });
    for (int o = 32; o > 0; o >>= 1)
      take(Candidate{__shfl_xor(best.total, o), static_cast<uint64_t>(__shfl_xor(static_cast<unsigned long long>(best.tie), o))});
    if (lane == 0) {
      sm_wtotal[wave] = best.total;
      sm_wtie[wave] = best.tie;
    }
    __syncthreads();
    for (int w = 0; w < kChooseWaves; ++w) take(Candidate{sm_wtotal[w], sm_wtie[w]});
    if (t == 0) put(r, best);
    last = best;
    __syncthreads();
  }
}

// Values a slice takes: wide ones where those already give the card's CUs a workgroup each.
int slice_values(int64_t rows, int32_t vocab) {
  return rows * ((vocab + kWideSlice - 1) / kWideSlice) >= 256 ? kWideSlice : kNarrowSlice;
}

int32_t slice_count(int64_t rows, int32_t vocab) {
  const int n = slice_values(rows, vocab);
  return (vocab + n - 1) / n;
}

}  // namespace
}  // namespace lkv

extern "C" int64_t lkv_beam_workspace_bytes(int32_t batch, int32_t beams, int32_t vocab, int32_t count) {
  using namespace lkv;
  if (batch <= 0 || beams <= 0 || vocab <= 0 || count <= 0) return 0;
  const int64_t rows = static_cast<int64_t>(batch) * beams;
  // (of up to 7 values more than the row has: the size that callers of this ABI version know)
  const int n = slice_values(rows, vocab);
  return rows * ((vocab + 7 + n - 1) / n) * (static_cast<int64_t>(sizeof(SliceSum)) + count * 8);
}

extern "C" int32_t lkv_beam_select(const lkv_beam_select_args* a, lkv_stream_t stream) {
  using namespace lkv;
  LKV_REQUIRE(a != nullptr, "null args");
  LKV_REQUIRE(a->struct_size == static_cast<int32_t>(sizeof(lkv_beam_select_args)),
              "lkv_beam_select_args size mismatch (caller %d, library %d)", a->struct_size,
              static_cast<int32_t>(sizeof(lkv_beam_select_args)));
  LKV_REQUIRE(a->batch >= 0, "bad sizes");
  LKV_REQUIRE(a->beams >= 1 && a->beams <= LKV_BEAM_MAX_BEAMS, "beams must be in [1, %d], got %d", LKV_BEAM_MAX_BEAMS, a->beams);
  LKV_REQUIRE(a->vocab >= 1 && a->vocab <= (1 << 20), "vocab must be in [1, 2^20], got %d", a->vocab);
  LKV_REQUIRE(a->count >= 1 && a->count <= LKV_BEAM_MAX_COUNT, "count must be in [1, %d], got %d", LKV_BEAM_MAX_COUNT, a->count);
  LKV_REQUIRE(a->logits_fp32 == 0 || a->logits_fp32 == 1, "logits_fp32 must be 0 or 1");
  if (a->batch == 0) return LKV_OK;  // (empty tensors have no address)
  LKV_REQUIRE(a->logits && a->scores && a->out_scores && a->out_beams && a->out_tokens, "null tensor");
  const int64_t rows = static_cast<int64_t>(a->batch) * a->beams;
  LKV_REQUIRE(rows <= 65535, "batch * beams must be <= 65535");
  LKV_REQUIRE((reinterpret_cast<uintptr_t>(a->logits) & (a->logits_fp32 ? 3 : 1)) == 0, "logits must be aligned to their type");
  const int64_t need = lkv_beam_workspace_bytes(a->batch, a->beams, a->vocab, a->count);
  if (a->workspace == nullptr || a->workspace_bytes < need)
    return fail(LKV_ERR_WORKSPACE, "beam selection needs %lld bytes of workspace, got %lld", static_cast<long long>(need),
                static_cast<long long>(a->workspace_bytes));
  LKV_REQUIRE((reinterpret_cast<uintptr_t>(a->workspace) & 15) == 0, "workspace must be 16-byte aligned");
  BeamParams p;
  p.logits = a->logits;
  p.sb = a->logits_stride_b;
  p.sk = a->logits_stride_k;
  p.scores = a->scores;
  p.scores_sb = a->scores_stride_b;
  p.out_scores = a->out_scores;
  p.out_beams = a->out_beams;
  p.out_tokens = a->out_tokens;
  p.beams = a->beams;
  p.vocab = a->vocab;
  p.count = a->count;
  p.slices = slice_count(rows, a->vocab);
  p.per_tile = 1.f / static_cast<float>((static_cast<int64_t>(p.slices) * a->count + 63) / 64);
  p.sums = static_cast<SliceSum*>(a->workspace);
  p.val = reinterpret_cast<float*>(p.sums + rows * p.slices);
  p.idx = reinterpret_cast<int32_t*>(p.val + rows * p.slices * a->count);
  const dim3 grid(p.slices, static_cast<unsigned>(rows));
  hipStream_t s = as_stream(stream);
  const bool wide = slice_values(rows, a->vocab) == kWideSlice;
  if (a->logits_fp32 && wide)
    beam_slice_kernel<true, kWideSlice / 4 / kBeamThreads><<<grid, kBeamThreads, 0, s>>>(p);
  else if (a->logits_fp32)
    beam_slice_kernel<true, kNarrowSlice / 4 / kBeamThreads><<<grid, kBeamThreads, 0, s>>>(p);
  else if (wide)
    beam_slice_kernel<false, kWideSlice / 8 / kBeamThreads><<<grid, kBeamThreads, 0, s>>>(p);
  else
    beam_slice_kernel<false, kNarrowSlice / 8 / kBeamThreads><<<grid, kBeamThreads, 0, s>>>(p);
  if (const int32_t st = check_launch("lkv_beam_select (slices)")) return st;
  beam_choose_kernel<<<a->batch, kChooseThreads, 0, s>>>(p);
  return check_launch("lkv_beam_select");
}
