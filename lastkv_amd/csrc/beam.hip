// Beam search's selection: the `count` best of a prompt's beams x vocab candidates score + (logit - lse(beam's logits)).
//
// Inside one beam the order of the totals is the order of the logits, so one pass over the logits does all of the reading:
//   slice kernel: a workgroup holds a slice of one beam's row in registers (8 to 32 values a thread), takes its maximum,
//     the sum of its exponentials and its `count` greatest logits;
//   choose kernel: a workgroup a prompt joins the slices' sums in 64 bits and chooses among the slices' candidates.
// Choosing the n greatest of many values needs no sort: the n-th greatest of the threads' own maxima is a floor that at
// least n values reach and few others do; those go to LDS and each counts the ones before it.  Where too many values reach
// the floor for LDS (equal logits), n rounds take the next one each; both give the same set.
// Bound by the read of the logits; small calls by two dependent launches.
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
// part of them).  64 groups are the fewest that do, and their counting the least: with groups of four the choice below,
// of 1024 threads, took 9.5 us in place of @@.
template <int kThreads>
struct FloorShared {
  float top[64];
  int32_t before[64];
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
  if (t % kGroup == 0) sm.top[t / kGroup] = x;
  if (part == 0) sm.before[i] = 0;
  __syncthreads();
  const float mine = sm.top[i];
  int before = 0;
#pragma unroll
  for (int j = part * kPart; j < (part + 1) * kPart; j += 4) {
    const float4 k = *reinterpret_cast<const float4*>(&sm.top[j]);
    before += (k.x > mine) || (k.x == mine && j < i);
    before += (k.y > mine) || (k.y == mine && j + 1 < i);
    before += (k.z > mine) || (k.z == mine && j + 2 < i);
    before += (k.w > mine) || (k.w == mine && j + 3 < i);
  }
  atomicAdd(&sm.before[i], before);
  __syncthreads();
  if (part == 0 && sm.before[i] == n - 1) sm.result = mine;
  __syncthreads();
  return sm.result;
}

// Eight bf16 or four fp32 values of a row from element e0 on; elements outside [0, V) are not read and become -inf.
template <bool kF32, int kVec>
__device__ inline void load_values(const void* row, int64_t e0, int V, float (&x)[kVec]) {
  if (e0 >= 0 && e0 + kVec <= V) {
    if constexpr (kF32) {
      const float4 f = *reinterpret_cast<const float4*>(static_cast<const float*>(row) + e0);
      x[0] = f.x;
      x[1] = f.y;
      x[2] = f.z;
      x[3] = f.w;
    } else {
      const uint4 w = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(row) + e0);
      const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        x[2 * j] = bf16_lo(u[j]);
        x[2 * j + 1] = bf16_hi(u[j]);
      }
    }
    return;
  }
#pragma unroll
  for (int j = 0; j < kVec; ++j) {
    const int64_t e = e0 + j;
    x[j] = kNegInf;
    if (e >= 0 && e < V)
      x[j] = kF32 ? static_cast<const float*>(row)[e] : bf16_bits_to_f32(static_cast<const uint16_t*>(row)[e]);
  }
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
  // 16-byte pieces start at addresses that are multiples of 16: the row's first piece may begin before it
  const int shift = static_cast<int>((reinterpret_cast<uintptr_t>(row) & 15) / (kF32 ? 4 : 2));
  const int e0 = (slice * kChunks * kBeamThreads + t) * kVec - shift;  // this thread's first element
  constexpr int kStep = kBeamThreads * kVec;
  float x[kChunks][kVec], top[kChunks];
#pragma unroll
  for (int c = 0; c < kChunks; ++c) load_values<kF32, kVec>(row, e0 + c * kStep, V, x[c]);
  if (t == 0) sm_n = 0;
  float best = kNegInf;  // (NaN where one is: its row then has no candidate, whatever the slices hold)
#pragma unroll
  for (int c = 0; c < kChunks; ++c) {
    top[c] = x[c][0];
#pragma unroll
    for (int j = 1; j + 1 < kVec; j += 2) top[c] = fmax3_nan(top[c], x[c][j], x[c][j + 1]);
    top[c] = fmax_nan(top[c], x[c][kVec - 1]);
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
  // the values that reach the floor, as (order, lowest index first)
  auto key = [&](float v, int e) {
    return (static_cast<uint64_t>(order_bits(v)) << 32) | static_cast<uint32_t>(~static_cast<uint32_t>(e));
  };
#pragma unroll
  for (int c = 0; c < kChunks; ++c) {
    if (!(top[c] >= floor && top[c] > kNegInf)) continue;
#pragma unroll
    for (int j = 0; j < kVec; ++j)
      if (x[c][j] >= floor && x[c][j] > kNegInf) {
        const uint32_t at = atomicAdd(&sm_n, 1u);
        if (at < kBeamCap) sm_cand[at] = key(x[c][j], e0 + c * kStep + j);
      }
  }
  const float ref = m == kNegInf ? 0.f : m;  // (x - ref is 0 for the greatest, whose term is then exactly 1)
  float part = 0.f;
#pragma unroll
  for (int c = 0; c < kChunks; ++c)
#pragma unroll
    for (int j = 0; j < kVec; ++j) part += fast_exp2((x[c][j] - ref) * kLog2e);  // (a +inf makes it NaN)
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
        if (!(x[c][j] > kNegInf)) continue;
        const uint64_t k = key(x[c][j], e0 + c * kStep + j);
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
  // the held tiles' tokens and logits are on their way while the sums are joined
  int token[kHeld];
  float logit[kHeld];
  auto fetch = [&](int tile, int& tk, float& x) {
    const int k = tile / tiles, i = (tile - k * tiles) * 64 + lane;
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
      if (m != to) s *= exp(static_cast<double>(m) - static_cast<double>(to));
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
    const int k = tile / tiles;
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
      const uint32_t at = atomicAdd(&sm_n, 1u);
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

// Slices of a row: its first 16-byte piece may hold up to 7 values that lie before the row.
int32_t slice_count(int64_t rows, int32_t vocab) {
  const int n = slice_values(rows, vocab);
  return (vocab + 7 + n - 1) / n;
}

}  // namespace
}  // namespace lkv

extern "C" int64_t lkv_beam_workspace_bytes(int32_t batch, int32_t beams, int32_t vocab, int32_t count) {
  using namespace lkv;
  if (batch <= 0 || beams <= 0 || vocab <= 0 || count <= 0) return 0;
  const int64_t rows = static_cast<int64_t>(batch) * beams;
  return rows * slice_count(rows, vocab) * (static_cast<int64_t>(sizeof(SliceSum)) + count * 8);
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
