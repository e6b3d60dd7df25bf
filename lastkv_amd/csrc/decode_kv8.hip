// Split-K decode attention over [8-bit shared pages | bf16 ring], also of a few query tokens a sequence.
//
// The scheme is the bf16 kernel's (decode.hip): a workgroup of 4 waves takes one (sequence, kv head, key split), a
// wave streams 32-token blocks from HBM to registers and keeps a running maximum, sum and O of its columns.  An older
// block is 8 KiB (K and V codes, 8 loads of 1 KiB) and two scale bytes; its codes become the exact bf16 operands of the bf16
// kernel (one conversion instruction for two values, the block's power of two applied by it), so that scores, softmax and
// sums are that kernel's, and with equal splits of an older segment alone the outputs are equal bit for bit.
#include "attn_common.h"
#include "common.h"
#include "decode_body.h"
#include "kv8.h"
#include "runtime.h"

namespace lkv {
namespace {

struct Block8 {
  uint4 k[4], v[4];
  uint32_t ks, vs;  // scale bytes
};

__device__ inline void load_block8(Block8& f, const Kv8Pool& o, int64_t base, int64_t sbase, int page, int lane) {
  const int64_t at = base + page * o.page + lane * 16;
#pragma unroll
  for (int i = 0; i < 4; ++i) f.k[i] = *reinterpret_cast<const uint4*>(o.k + at + i * 1024);
#pragma unroll
  for (int i = 0; i < 4; ++i) f.v[i] = *reinterpret_cast<const uint4*>(o.v + at + i * 1024);
  f.ks = o.ks[sbase + page];
  f.vs = o.vs[sbase + page];
}

// Bytes of the first n (of four) tokens of a word.
__device__ inline uint32_t keep_bytes(uint32_t w, int n) {
  return n >= 4 ? w : n <= 0 ? 0u : w & ((1u << (8 * n)) - 1u);
}

// The bf16 operands of a block whose first `hi` tokens count (V codes of the others become 0: they may be anything, and 0 * NaN is NaN).
__device__ inline void expand_block8(const Block8& f, int hi, int g4, BlockFrags& x) {
  const float ks = kv8_scale(f.ks), vs = kv8_scale(f.vs);
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
    x.v[2 * i] = kv8_to_bf16(c.x, c.y, vs);
    x.v[2 * i + 1] = kv8_to_bf16(c.z, c.w, vs);
  }
}

template <bool kVScale, bool kMulti, int CG, bool kPairs>
__global__ __launch_bounds__(256) void decode_kv8_kernel(const DecodeParams p, const Kv8Pool o) {
  __shared__ DecodeShared<CG> sm;
  DecodeItem it;
  if (!decode_item<kMulti>(p, blockIdx.x, it)) return;  // (workgroup-uniform)
  constexpr int kStride = kPairs ? 2 : kDecodeWaves;    // block stride of one wave
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n16 = lane & 15, g4 = lane >> 4;
  const int G = p.group, kvh = it.kvh, b = it.b;
  const int Lq = it.mr.L;
  const SeqView sv = make_seq_view(p.seg, b, kvh);
  const int nbl = local_blocks(sv, sv.n1);
  // The split's share in bytes: an older block counts 1, a ring block 2.
  const int units = sv.nb0 + 2 * nbl, per = (units + it.S - 1) / it.S;
  const int u0 = min(it.split * per, units), u1 = min(u0 + per, units);
  const int ob = min(u0, sv.nb0), oe = min(u1, sv.nb0);
  const int lb = sv.nb0 + ((max(u0 - sv.nb0, 0) + 1) >> 1), le = sv.nb0 + ((max(u1 - sv.nb0, 0) + 1) >> 1);

  const int cols = kMulti ? G * Lq : G;
  uint4 qf[CG][4];
  int lim[CG], lim_min = 0;  // causal limits (local token index) of this lane's columns and of column 0
  if (kMulti) lim_min = p.causal ? sv.n1 - Lq : sv.n1 - 1;
  const int cg0 = kPairs ? (wave >> 1) * CG : 0;
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
  const float vs = kVScale ? p.vscale[kvh] : 1.f;
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
      compute_block<kVScale, kMulti>(f, r, qf[cg], vs, p.scale_log2, n16, g4, lim[cg], lim_min, st[cg]);
  };
  const int w = kPairs ? (wave & 1) : wave;

  // older blocks: ob + w, + kStride, ...
  const int64_t base = kvh * o.hs, sbase = kvh * o.s_hs;
  uint32_t nan = 0;  // a NaN block was among them
  auto page = [&](int blk) { return min(max(sv.otab[blk], 0), o.pages - 1); };
  auto compute8 = [&](const Block8& f, int blk) __attribute__((always_inline)) {
    BlockRef r;
    r.lo = 0;
    r.hi = min(kBlockTokens, sv.n0 - blk * kBlockTokens);
    r.seg_tok = -1;
    r.older = true;
    nan |= (f.ks == 255u) | (f.vs == 255u);
    BlockFrags x;
    expand_block8(f, r.hi, g4, x);
    compute(x, r);
  };
  int blk = ob + w;
  if (blk < oe) {
    Block8 fa, fb;
    load_block8(fa, o, base, sbase, page(blk), lane);
    while (blk + kStride < oe) {
      load_block8(fb, o, base, sbase, page(blk + kStride), lane);
      __builtin_amdgcn_sched_barrier(0);
      compute8(fa, blk);
      blk += kStride;
      fa = fb;
    }
    compute8(fa, blk);
  }
  // ring blocks: lb + w, + kStride, ...
  blk = lb + w;
  if (blk < le) {
    BlockFrags fa, fb;
    BlockRef ra = block_ref(sv, blk), rb;
    load_block<false>(fa, ra, n16, g4);
    while (blk + kStride < le) {
      rb = block_ref(sv, blk + kStride);
      load_block<false>(fb, rb, n16, g4);
      __builtin_amdgcn_sched_barrier(0);
      compute(fa, ra);
      blk += kStride;
      fa = fb;
      ra = rb;
    }
    compute(fa, ra);
  }
  if (nan) {
#pragma unroll
    for (int cg = 0; cg < CG; ++cg) st[cg].l = __builtin_nanf("");
  }
  decode_merge_waves<kMulti, CG, kPairs, true>(p, it, st, sm);
}

template <int CG, bool kPairs>
void launch_multi8(const DecodeParams& p, const Kv8Pool& o, dim3 grid, bool vscale, hipStream_t s) {
  if (vscale)
    decode_kv8_kernel<true, true, CG, kPairs><<<grid, 256, 0, s>>>(p, o);
  else
    decode_kv8_kernel<false, true, CG, kPairs><<<grid, 256, 0, s>>>(p, o);
}

}  // namespace

void launch_decode_kv8(const DecodeParams& p, const Kv8Pool& older, dim3 grid, bool vscale, int cg, hipStream_t s) {
  if (cg == 1)
    launch_multi8<1, false>(p, older, grid, vscale, s);
  else if (cg == 2)
    launch_multi8<2, false>(p, older, grid, vscale, s);
  else if (cg == 4)
    launch_multi8<2, true>(p, older, grid, vscale, s);
  else if (vscale)
    decode_kv8_kernel<true, false, 1, false><<<grid, 256, 0, s>>>(p, older);
  else
    decode_kv8_kernel<false, false, 1, false><<<grid, 256, 0, s>>>(p, older);
}

}  // namespace lkv
