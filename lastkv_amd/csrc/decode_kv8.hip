// Split-K decode attention over [8-bit shared pages | bf16 ring], also of a few query tokens a sequence.
//
// The scheme is the bf16 kernel's (decode.hip): a workgroup takes one (sequence, kv head, key split), a
// wave streams 32-token blocks from HBM to registers and keeps a running maximum, sum and O of its columns.  An older
// block is 8 KiB (K and V codes, 8 loads of 1 KiB) and two scale bytes; its codes become the exact bf16 operands of the bf16
// kernel (one conversion instruction for two values, the block's power of two applied by it), so that scores, softmax and
// sums are that kernel's.
//
// Bound by memory for many rows (32 sequences of 9.2K keys, 8 kv heads: 105 us, 6.5 TB/s; 4 of 128K 175 us, 6.2; the bf16 kernel's
// calls 178 and 328), for few by the blocks that follow each other in a wave (7 sequences of up to 12K keys, 4 kv heads, s per
// head: 15-18 us where the bytes are 4).  Half the bytes a block ask for twice the blocks in flight: eight waves of three
// buffers, so that two blocks are on their way while one is computed, and nothing but the blocks goes through vector loads (32
// sequences 126 us with two buffers and page ids and scales by vector loads).  Dealing the blocks to all waves of all splits,
// with a pair's splits on one XCD, reads one window at a time: 6.6-6.8 TB/s where a range a split reads 5.8.
#include "attn_common.h"
#include "common.h"
#include "decode_body.h"
#include "kv8.h"
#include "runtime.h"

namespace lkv {
namespace {

// Waves of a workgroup: two a SIMD, one for two column groups (whose state takes more than half of a SIMD's registers).
constexpr int waves8(int cg) { return cg == 1 ? 8 : 4; }

typedef const __attribute__((address_space(4))) uint32_t* ConstWords;

// Words of constant memory: what is the same for a wave is then read with scalar loads, whose waits leave the blocks' vector
// loads in flight.
__device__ inline ConstWords const_words(const void* p) { return (ConstWords)p; }

struct Block8 {
  uint4 k[4], v[4];
  uint32_t ks, vs, page;  // the words that hold the page's scale bytes

  __device__ uint32_t byte(uint32_t w) const { return (w >> (8 * (page & 3))) & 0xffu; }
};

template <bool kNT>
__device__ inline uint4 load16(const uint8_t* p) {
  return kNT ? load_nt(p) : *reinterpret_cast<const uint4*>(p);
}

// The pool's part of one kv head.
struct HeadPool {
  const uint8_t* k;
  const uint8_t* v;
  ConstWords ks, vs;
  int64_t page;
  int32_t pages;
};

__device__ inline HeadPool head_pool(const Kv8Pool& o, int kvh) {
  return HeadPool{o.k + kvh * o.hs, o.v + kvh * o.hs, const_words(o.ks + kvh * o.s_hs), const_words(o.vs + kvh * o.s_hs), o.page, o.pages};
}

template <bool kNT>
__device__ inline void load_block8(Block8& f, const HeadPool& o, int page, int lane) {
  const int64_t at = page * o.page + lane * 16;
#pragma unroll
  for (int i = 0; i < 4; ++i) f.k[i] = load16<kNT>(o.k + at + i * 1024);
#pragma unroll
  for (int i = 0; i < 4; ++i) f.v[i] = load16<kNT>(o.v + at + i * 1024);
  f.ks = o.ks[page >> 2];
  f.vs = o.vs[page >> 2];
  f.page = page;
}

// Bytes of the first n (of four) tokens of a word.
__device__ inline uint32_t keep_bytes(uint32_t w, int n) {
  return n >= 4 ? w : n <= 0 ? 0u : w & ((1u << (8 * n)) - 1u);
}

// Eight codes times a power of two, in fp32 exactly, and then times s, rounded to bf16: bf16(value * s).  (The power of two times s first
// may lie beyond fp32 where no value does, and would turn the block's zeros into NaN.)
__device__ inline uint4 scaled_to_bf16(uint32_t lo, uint32_t hi, float scale, float s) {
  const auto a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(lo, scale, false), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(lo, scale, true);
  const auto c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(hi, scale, false), d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(hi, scale, true);
  return make_uint4(pack_bf16x2(a[0] * s, a[1] * s), pack_bf16x2(b[0] * s, b[1] * s), pack_bf16x2(c[0] * s, c[1] * s),
                    pack_bf16x2(d[0] * s, d[1] * s));
}

// The bf16 operands of a block whose first `hi` tokens count (V codes of the others become 0: they may be anything, and 0 * NaN is
// NaN); kVScale: V times s.
template <bool kVScale>
__device__ inline void expand_block8(const Block8& f, int hi, int g4, float s, BlockFrags& x) {
  const float ks = kv8_scale(f.byte(f.ks)), vs = kv8_scale(f.byte(f.vs));
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x.k[i >> 1][2 * (i & 1)] = kv8_to_bf16(f.k[i].x, f.k[i].y, ks);
    x.k[i >> 1][2 * (i & 1) + 1] = kv8_to_bf16(f.k[i].z, f.k[i].w, ks);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint4 c = f.v[i];
    if (hi < kBlockTokens) {
      const int n = hi - 8 * g4;
      c = make_uint4(keep_bytes(c.x, n), keep_bytes(c.y, n - 4), keep_bytes(c.z, n), keep_bytes(c.w, n - 4));
    }
    x.v[2 * i] = kVScale ? scaled_to_bf16(c.x, c.y, vs, s) : kv8_to_bf16(c.x, c.y, vs);
    x.v[2 * i + 1] = kVScale ? scaled_to_bf16(c.z, c.w, vs, s) : kv8_to_bf16(c.z, c.w, vs);
  }
}

// The kernel's arguments, read again where they are needed: held from its start, with those of the other segment and of
// the merge, they take more scalar registers than there are.
struct Arguments {
  DecodeParams p;
  Kv8Pool o;
};

__device__ inline const Arguments& reread() {
  uint32_t zero;
  asm volatile("s_mov_b32 %0, 0" : "=s"(zero));
  typedef const __attribute__((address_space(4))) uint8_t* Kernarg;
  return *reinterpret_cast<const Arguments*>((const uint8_t*)((Kernarg)__builtin_amdgcn_kernarg_segment_ptr() + zero));
}

template <bool kVScale, bool kNT, bool kMulti, int CG, bool kPairs>
__global__ __launch_bounds__(waves8(CG) * 64, waves8(CG) / 4) void decode_kv8_kernel(const Arguments args) {
  const DecodeParams& p = args.p;
  constexpr int kWaves = waves8(CG);
  constexpr int kStride = kPairs ? kWaves / 2 : kWaves;  // waves that share the blocks of a workgroup
  __shared__ DecodeShared<CG, kWaves> sm;
  DecodeItem it;
  if (!decode_item<kMulti>(p, blockIdx.x, it)) return;  // (workgroup-uniform)
  // The splits of one (sequence, kv head) side by side on one XCD, the heads of one sequence apart: a long sequence among short
  // ones keeps all XCDs busy (8 sequences, one of 9000 tokens and the others below 1000: 22.7 us, with its heads side by side 28.9;
  // equal lengths as before, 24 of 9300 77 where it was 84).  An XCD takes another head of each sequence: with the same one
  // of all 64 of 9300 tokens took 219 us, so 210.
  if (p.cu == nullptr) {
    const int id = blockIdx.x + gridDim.x * (blockIdx.y + gridDim.y * blockIdx.z);
    const int at = xcd_logical_index(id, gridDim.x * gridDim.y * gridDim.z);
    it.split = at % it.S;
    it.b = at / it.S % gridDim.z;
    it.kvh = (at / (it.S * gridDim.z) + it.b) % gridDim.y;
    it.mr = kMulti ? multi_rows(p, it.b) : MultiRows{1, it.b};
    it.ws_row0 = it.mr.row0;
  }
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n16 = lane & 15, g4 = lane >> 4;
  const int G = p.group, kvh = it.kvh, b = it.b;
  const int Lq = it.mr.L;
  const int cols = kMulti ? G * Lq : G;
  const SeqView sv = make_seq_view(p.seg, b, kvh);
  uint4 qf[CG][4];
  int lim[CG], lim_min = 0;  // causal limits (local token index) of this lane's columns and of column 0
  if (kMulti) lim_min = p.causal ? sv.n1 - Lq : sv.n1 - 1;
  const int cg0 = kPairs ? wave / kStride * CG : 0;
#pragma unroll
  for (int cg = 0; cg < CG; ++cg) {
    const int c = 16 * (cg0 + cg) + n16;
    const int t = kMulti ? c / G : 0, h = c - t * G;
    const uint16_t* qrow = p.q + (kMulti && p.cu ? it.mr.row0 * p.q_st : b * p.q_sb) + (kMulti ? t * p.q_st : 0) +
                           static_cast<int64_t>(kvh * G + h) * kHeadDim;
#pragma unroll
    for (int kb = 0; kb < 4; ++kb)
      qf[cg][kb] = c < cols ? *reinterpret_cast<const uint4*>(qrow + 32 * kb + 8 * g4) : make_uint4(0, 0, 0, 0);
    lim[cg] = kMulti && p.causal ? lim_min + t : lim_min;
  }
  const float vs = kVScale ? p.vscale[kvh] : 1.f, scale_log2 = p.scale_log2;
  SoftmaxState st[CG];
#pragma unroll
  for (int cg = 0; cg < CG; ++cg) {
    st[cg].m = kDecodeNegInf;
    st[cg].l = 0.f;
#pragma unroll
    for (int nb = 0; nb < 8; ++nb) st[cg].o[nb] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  auto compute = [&](const BlockFrags& f, const BlockRef& r) __attribute__((always_inline)) {
#pragma unroll
    for (int cg = 0; cg < CG; ++cg)
      compute_block<false, kMulti>(f, r, qf[cg], 1.f, scale_log2, n16, g4, lim[cg], lim_min, st[cg]);
  };

  // The blocks of a segment are dealt one by one to all waves of all splits, so that the workgroups of a (sequence, kv head)
  // walk one window of its K and V together; the waves that got one ring block less have the first older ones.
  const int me = it.split * kStride + (kPairs ? wave % kStride : wave), step = it.S * kStride;
  const int nbl = local_blocks(sv, sv.n1), nb0 = sv.nb0, n0 = sv.n0;
  int first = me - nbl % step;
  if (first < 0) first += step;
  const int n = first < nb0 ? (nb0 - 1 - first) / step + 1 : 0;
  uint32_t nan = 0;  // a NaN block was among them
  const ConstWords table = const_words(sv.otab);
  HeadPool o;
  Block8 f0, f1, f2;
  int pg = 0;
  // With few pairs the heads start their walks apart: heads and sequences whose pages lie a power of two from each other would be read at
  // the same place of all of them, and so from the same memory channels (replayed calls over 4 sequences of 131072 tokens: 205 us
  // where all start at 0, 186 so; 2 sequences 115 and 104; other lengths and more pairs within 3 %).  The start goes by the
  // head and the sequence's own length alone, so that with a fixed split count a sequence's bits do not depend on its place in
  // the batch (starts that differ by sequence too: 183).
  const int apart = it.S < 4 ? 0 : nb0 >= 1024 ? 1023 : nb0 >= 256 ? 255 : 0;
  const int rot = (kvh * 101) & apart;
  auto at = [&](int t) {
    const int i = first + step * t + rot;
    return i >= nb0 ? i - nb0 : i;
  };
  auto look = [&](int t) { pg = min(max(static_cast<int>(table[at(min(t, n - 1))]), 0), o.pages - 1); };
  auto load = [&](Block8& f) __attribute__((always_inline)) { load_block8<kNT>(f, o, pg, lane); };
  auto compute8 = [&](const Block8& f, int t) __attribute__((always_inline)) {
    BlockRef r;
    r.lo = 0;
    r.hi = min(kBlockTokens, n0 - at(t) * kBlockTokens);
    r.seg_tok = -1;
    r.older = true;
    nan |= static_cast<uint32_t>(f.byte(f.ks) == 255u || f.byte(f.vs) == 255u);
    BlockFrags x;
    expand_block8<kVScale>(f, r.hi, g4, vs, x);
    compute(x, r);
  };
  // The first two older blocks are on their way while the last ring block is computed.
  auto begin = [&]() __attribute__((always_inline)) {
    if (n == 0) return;
    o = head_pool(reread().o, kvh);
    look(0);
    load(f0);
    if (n == 1) return;
    look(1);
    load(f1);
    look(2);
  };
  int blk = nb0 + me;
  const int le = nb0 + nbl;
  BlockFrags fa, fb;
  BlockRef ra, rb;
  const bool ring = blk < le;
  if (ring) {
    ra = block_ref(sv, blk);
    load_block<kNT>(fa, ra, n16, g4);
    while (blk + step < le) {
      rb = block_ref(sv, blk + step);
      load_block<kNT>(fb, rb, n16, g4);
      __builtin_amdgcn_sched_barrier(0);
      compute(fa, ra);
      blk += step;
      fa = fb;
      ra = rb;
    }
  }
  begin();
  __builtin_amdgcn_sched_barrier(0);
  if (ring) compute(fa, ra);
  if (n > 0) {
    // Two blocks are on their way while one is computed.  In the loop the loads are unconditional (the compiler
    // then counts them exactly for its waits), and the page of the next one is looked up a step ahead.
    int t = 0;
    auto pass = [&](Block8& in, const Block8& now, int i) __attribute__((always_inline)) {
      load(in);
      look(t + i + 3);
      __builtin_amdgcn_sched_barrier(0);
      compute8(now, t + i);
      __builtin_amdgcn_sched_barrier(0);
    };
    for (; t + 4 < n; t += 3) {
      pass(f2, f0, 0);
      pass(f0, f1, 1);
      pass(f1, f2, 2);
    }
    // one to four are left, two of them loaded
    if (t + 2 < n) load(f2);
    compute8(f0, t);
    if (t + 3 < n) {
      look(t + 3);
      load(f0);
    }
    if (t + 1 < n) compute8(f1, t + 1);
    if (t + 2 < n) compute8(f2, t + 2);
    if (t + 3 < n) compute8(f0, t + 3);
  }
  if (nan) {
#pragma unroll
    for (int cg = 0; cg < CG; ++cg) st[cg].l = __builtin_nanf("");
  }
  decode_merge_waves<kMulti, CG, kPairs, true, kWaves>(reread().p, it, st, sm);
}

template <bool kMulti, int CG, bool kPairs>
void launch8(const DecodeParams& p, const Kv8Pool& o, dim3 grid, bool vscale, bool nt, hipStream_t s) {
  if (vscale && nt)
    decode_kv8_kernel<true, true, kMulti, CG, kPairs><<<grid, waves8(CG) * 64, 0, s>>>(Arguments{p, o});
  else if (vscale)
    decode_kv8_kernel<true, false, kMulti, CG, kPairs><<<grid, waves8(CG) * 64, 0, s>>>(Arguments{p, o});
  else if (nt)
    decode_kv8_kernel<false, true, kMulti, CG, kPairs><<<grid, waves8(CG) * 64, 0, s>>>(Arguments{p, o});
  else
    decode_kv8_kernel<false, false, kMulti, CG, kPairs><<<grid, waves8(CG) * 64, 0, s>>>(Arguments{p, o});
}

}  // namespace

void launch_decode_kv8(const DecodeParams& p, const Kv8Pool& older, dim3 grid, bool vscale, bool nt, int cg, hipStream_t s) {
  if (cg == 1)
    launch8<true, 1, false>(p, older, grid, vscale, nt, s);
  else if (cg == 2)
    launch8<true, 2, false>(p, older, grid, vscale, nt, s);
  else if (cg == 4)
    launch8<true, 2, true>(p, older, grid, vscale, nt, s);
  else
    launch8<false, 1, false>(p, older, grid, vscale, nt, s);
}

}  // namespace lkv
