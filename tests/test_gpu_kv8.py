"""The shared cache in 8 bits: quantisation, and the attention that reads it, against 64-bit forms (gpu)."""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from lastkv_amd import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16 = torch.bfloat16


# ---------------------------------------------------------------------------------------- references
def grid():
    """The non-negative e4m3 values, in order."""

    v = [m * 2.0 ** -9 for m in range(8)] + [(8 + m) / 8 * 2.0 ** e for e in range(-6, 9) for m in range(8)]
    return np.array([x for x in v if x <= 448.0])


def quantized(x):
    """float64 [..., 32, 128] blocks -> (their values after quantisation, scale exponents); NaN blocks are NaN."""

    g = grid()
    mids = (g[1:] + g[:-1]) / 2
    powers = 2.0 ** np.arange(-127, 128)
    amax = np.abs(x).max((-2, -1), keepdims=True)
    bad = ~np.isfinite(amax)
    scale = powers[np.minimum(np.searchsorted(448.0 * powers, np.where(bad, 0, amax)), 254)]  # the first that holds amax
    v = np.abs(np.where(bad, 0, x)) / scale
    lo, hi = np.searchsorted(mids, v, side="left"), np.searchsorted(mids, v, side="right")
    y = np.sign(np.where(bad, 0, x)) * g[np.where(lo % 2 == 0, lo, hi)] * scale
    return np.where(bad, np.nan, y), scale


def blocks_of(x, tokens):
    """[T, 128] rows as [nb, 32, 128] blocks, zero past the end."""

    nb = -(-tokens // 32)
    out = np.zeros((nb * 32, 128))
    out[:tokens] = x[:tokens]
    return out.reshape(nb, 32, 128)


def rand(seed, *shape, gain=True):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=g)
    if gain:
        x = x * torch.exp(0.4 * torch.randn(shape[-1], generator=g))
    return x.to(BF16)


def table_of(B, W, seed=None, first=0):
    ids = np.arange(first, first + B * W)
    if seed is not None:
        ids = np.random.default_rng(seed).permutation(ids)
    return torch.from_numpy(ids.reshape(B, W).astype(np.int32)).to(DEV)


def paged(k, v, table, pages=None, token0=0, wrap=0):
    """[B, T, H, 128] rows in a bf16 pool."""

    pool = ops.PagedKV.zeros(pages or table.numel(), k.shape[2], DEV)
    ops.append_paged(k.to(DEV), v.to(DEV), pool, table, token0=token0, wrap_tokens=wrap)
    return pool


def history(seed, B, H, T, shuffle=True, spare=0):
    """An 8-bit pool of T tokens a sequence in pages of any order: (pool, table, values K, values V [B, H, T, 128])."""

    W = max(1, -(-T // 32))
    table = table_of(B, W, seed if shuffle else None, first=spare)
    k, v = rand(seed, B, W * 32, H, 128), rand(seed + 1, B, W * 32, H, 128)
    src = paged(k, v, table, pages=B * W + spare)
    pool = ops.PagedKV8.zeros(B * W + spare, H, DEV)
    ops.kv8_quantize(src, pool, src_table=table, dst_table=table, tokens=W * 32)
    kv = ops.kv8_unpack(pool, table, 0, W * 32)
    return pool, table, kv[0], kv[1]


# ---------------------------------------------------------------------------------------- quantisation
@pytest.mark.parametrize("B,H,T,first", [(1, 1, 1, 0), (2, 3, 33, 0), (3, 2, 64, 1), (1, 8, 95, 1), (2, 1, 31, 0)])
def test_quantize_is_the_formula_bit_for_bit(B, H, T, first):
    k, v = rand(T, B, T, H, 128), rand(T + 1, B, T, H, 128)
    W = -(-T // 32) + 1
    st, dt = table_of(B, W, 5), table_of(B, W, 6, first=2)
    src = paged(k, v, st)
    dst = ops.PagedKV8.zeros(B * W + 2, H, DEV)
    dst.k.view(torch.uint8).fill_(0x55)
    dst.v.view(torch.uint8).fill_(0x55)
    dst.k_scales.fill_(99)
    ops.kv8_quantize(src, dst, src_table=st, dst_table=dt, tokens=T, first_block=first)
    written = {int(p) for p in dt[:, first:-(-T // 32)].flatten()}
    for p in range(dst.pages):  # nothing else is touched
        if p not in written:
            assert bool((dst.k[:, p].view(torch.uint8) == 0x55).all()) and bool((dst.k_scales[:, p] == 99).all())
    got = ops.kv8_unpack(dst, dt, 32 * first, T - 32 * first)
    for x, y, sc in ((k, got[0], dst.k_scales), (v, got[1], dst.v_scales)):
        for b in range(B):
            for h in range(H):
                want, scale = quantized(blocks_of(x[b, :, h].double().numpy(), T))
                have = y[b, h].double().cpu().numpy()
                assert np.array_equal(have, want.reshape(-1, 128)[32 * first:T])
                e = sc[h, dt[b, first:-(-T // 32)].long()].cpu().numpy().astype(float)
                assert np.array_equal(2.0 ** (e - 127), scale.reshape(-1)[first:])


def test_quantize_every_bf16_value_and_border():
    """Blocks of one magnitude each: every bf16 value of some exponents next to 448 times a power of two, and the ends of the range."""

    bits = np.concatenate([np.arange(e << 7, (e + 1) << 7) for e in (0, 1, 2, 7, 8, 9, 20, 126, 127, 200, 253, 254)])
    x = torch.from_numpy(bits.astype(np.int16)).view(BF16)
    T = 32 * len(bits)
    k = torch.zeros(T, 128)
    for i, val in enumerate(x.float()):  # the block's greatest value, and fractions of it down to nothing
        k[32 * i:32 * i + 32] = val * 2.0 ** -torch.arange(32.)[:, None] * torch.linspace(-1, 1, 128)
        k[32 * i, 0] = val
    k = k.to(BF16)[None, :, None]
    table = table_of(1, T // 32)
    pool = ops.PagedKV8.zeros(T // 32, 1, DEV)
    ops.kv8_quantize(paged(k, k, table), pool, src_table=table, dst_table=table, tokens=T)
    got, _ = ops.kv8_unpack(pool, table, 0, T)
    want, _ = quantized(blocks_of(k[0, :, 0].double().numpy(), T))
    want = torch.from_numpy(want.reshape(T, 128)).float().to(BF16)  # (below bf16's least subnormal value the unpacked one is rounded)
    assert torch.equal(got[0, 0].cpu(), want)


@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
def test_a_block_with_an_infinity_or_nan_is_nan_and_no_other(bad):
    k, v = rand(1, 1, 96, 2, 128), rand(2, 1, 96, 2, 128)
    k[0, 40, 1, 7] = bad
    v[0, 95, 0, 127] = bad  # (the last token, left out below)
    table = table_of(1, 3)
    pool = ops.PagedKV8.zeros(3, 2, DEV)
    ops.kv8_quantize(paged(k, v, table), pool, src_table=table, dst_table=table, tokens=95)
    assert pool.k_scales.eq(255).nonzero().tolist() == [[1, 1]] and not bool(pool.v_scales.eq(255).any())
    gk, gv = ops.kv8_unpack(pool, table, 0, 95)
    assert bool(gk[0, 1, 32:64].isnan().all()) and int(gk.isnan().sum()) == 32 * 128 and not bool(gv.isnan().any())


def test_quantize_takes_device_lengths_and_leaves_later_blocks():
    B, H, W = 4, 2, 3
    k, v = rand(3, B, 96, H, 128), rand(4, B, 96, H, 128)
    table = table_of(B, W, 1)
    src = paged(k, v, table)
    lens = torch.tensor([0, 1, 64, 500], dtype=torch.int32, device=DEV)
    a, b = (ops.PagedKV8.zeros(B * W, H, DEV) for _ in range(2))
    ops.kv8_quantize(src, a, src_table=table, dst_table=table, tokens=lens)
    for i, n in enumerate([0, 1, 64, 96]):
        if n:
            ops.kv8_quantize(src, b, src_table=table[i:i + 1], dst_table=table[i:i + 1], tokens=n)
    for x, y in ((a.k, b.k), (a.v, b.v), (a.k_scales, b.k_scales), (a.v_scales, b.v_scales)):
        assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))


def test_quantizing_the_values_again_keeps_them():
    pool, table, k, v = history(9, 2, 3, 100)
    again = ops.PagedKV8.zeros(pool.pages, 3, DEV)
    ops.kv8_quantize(paged(k.transpose(1, 2), v.transpose(1, 2), table), again, src_table=table, dst_table=table, tokens=128)
    k2, v2 = ops.kv8_unpack(again, table, 0, 128)
    assert torch.equal(k, k2) and torch.equal(v, v2)


# ---------------------------------------------------------------------------------------- attention
def attention64(q, k, v, own):
    """[L, Hq, 128] over [Hkv, T, 128], the last `own` keys being the queries'; (out, mean |v| under the weights, bound of a
    score's error) in 64 bits.  A score is a sum of 128 products in fp32, with an error of at most 130 * 2^-24 of the sum of
    their magnitudes."""

    L, Hq, _ = q.shape
    H, T, _ = k.shape
    q = q.double().view(L, H, Hq // H, 128).permute(1, 2, 0, 3)
    k, v = k.double(), v.double()
    if T == 0:
        z = torch.zeros(L, Hq, 128, dtype=torch.float64)
        return z, z, 0.0, torch.full((L, Hq), -math.inf, dtype=torch.float64)
    s = q @ k.transpose(1, 2)[:, None] / math.sqrt(128)
    err = float((q.abs() @ k.abs().transpose(1, 2)[:, None]).max()) / math.sqrt(128) * 130 * 2.0 ** -24
    hidden = torch.arange(T)[None, :] > (T - own + torch.arange(L))[:, None]
    s = s.masked_fill(hidden, -math.inf) if own else s
    p = torch.softmax(s, -1)
    back = lambda x: x.permute(2, 0, 1, 3).reshape(L, Hq, 128)
    return back(p @ v[:, None]), back(p @ v.abs()[:, None]), err, torch.logsumexp(s, -1).permute(2, 0, 1).reshape(L, Hq)


def check(got, want, mean, err, p_err, what=""):
    """bf16's rounding (2^-8 of the value), and weights off by the scores' error (twice: weight and sum) and by p_err."""

    off = (got.double().cpu() - want).abs()
    room = want.abs() * 2.0 ** -8 + mean * (2 * err + p_err) + 1e-30
    worst = float((off / room).max())
    assert worst <= 1, (what, worst)


SEG = [  # (Hq, Hkv, older, local, vscale)
    (8, 2, [0, 1, 31, 33, 700], [1, 40, 0, 64, 7], True),
    (32, 8, [2048, 2047, 2049], [3, 100, 1], False),
    (28, 4, [130, 0, 0], [0, 0, 96], True),
    (5, 5, [64], [33], True),
    (64, 4, [257, 96], [5, 1], False),   # 16 heads a kv head
    (40, 2, [300, 70], [31, 5], True),   # 20: two column groups
    (64, 1, [300, 70], [31, 5], False),  # 64: four
]


def segments(seed, Hq, Hkv, older, local, vscale, ring_blocks=4, shuffle=True):
    """Arguments of a call over [8-bit history | bf16 ring] and what a 64-bit form needs."""

    B = len(older)
    pool, table, k8, v8 = history(seed, B, Hkv, max(max(older), 1), shuffle)
    ring_tokens = 32 * ring_blocks
    kl, vl = rand(seed + 2, B, ring_tokens, Hkv, 128), rand(seed + 3, B, ring_tokens, Hkv, 128)
    rtab = table_of(B, ring_blocks, seed + 4)
    ring = ops.PagedKV.zeros(rtab.numel(), Hkv, DEV)
    for b in range(B):
        if local[b]:
            ops.append_paged(kl[b:b + 1, :local[b]].to(DEV), vl[b:b + 1, :local[b]].to(DEV), ring, rtab[b:b + 1],
                             token0=older[b], wrap_tokens=ring_tokens)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)
    vs = (torch.rand(Hkv, generator=torch.Generator().manual_seed(seed)) + 0.5).to(BF16).float().to(DEV) if vscale else None
    seg = dict(older=pool, older_table=table, older_len=i32(older), vscale=vs, local=ring, local_table=rtab,
               local_ring_blocks=ring_blocks, local_len=i32(local), local_start=i32([n % ring_tokens for n in older]))
    vh = v8 if vs is None else (v8.float() * vs[:, None, None]).to(BF16)
    keys = []
    for b in range(B):
        cat = lambda h, l: torch.cat((h[b, :, :older[b]].cpu(), l[b, :local[b]].transpose(0, 1)), 1)
        keys.append((cat(k8, kl), cat(vh, vl)))
    return seg, keys


@pytest.mark.parametrize("splits", [None, 1, 3])
@pytest.mark.parametrize("Hq,Hkv,older,local,vscale", SEG)
def test_decode_against_64_bits(Hq, Hkv, older, local, vscale, splits):
    seg, keys = segments(11, Hq, Hkv, older, local, vscale)
    B = len(older)
    q = rand(17, B, Hq, 128, gain=False)
    lse = torch.empty(B, Hq, device=DEV)
    out = ops.decode_attention(q.to(DEV), num_splits=splits, lse=lse, **seg)
    for b, (k, v) in enumerate(keys):
        want, mean, err, wl = attention64(q[b:b + 1], k, v, 0)
        check(out[b:b + 1], want, mean, err, 2.0 ** -15, (b, splits))  # (a weight is carried as two bf16: 2^-17, and exp2, and sums)
        if older[b] + local[b] == 0:
            assert bool((out[b] == 0).all()) and bool((lse[b] == -math.inf).all())
        else:
            assert float((lse[b].double().cpu() - wl[0]).abs().max()) <= err + 2.0 ** -20 * (1 + float(wl.abs().max()))


@pytest.mark.parametrize("splits", [1, 2, 5])
@pytest.mark.parametrize("vscale", [False, True])
@pytest.mark.parametrize("T", [1, 32, 100])
def test_decode_over_a_history_alone_is_the_bf16_call_over_its_values(T, vscale, splits):
    """A block a wave, joined in the same order: equal in every bit."""

    pool, table, k, v = history(T, 3, 4, T)
    twin = paged(k.transpose(1, 2), v.transpose(1, 2), table)
    q = rand(5, 3, 16, 128, gain=False).to(DEV)
    vs = torch.tensor([0.5, 1.25, -2.0, 0.7], device=DEV).to(BF16).float() if vscale else None
    lens = torch.tensor([T, T // 2, 0], dtype=torch.int32, device=DEV)
    for n in (T, lens):
        a = ops.decode_attention(q, older=pool, older_table=table, older_len=n, vscale=vs, num_splits=splits)
        b = ops.decode_attention(q, older=twin, older_table=table, older_len=n, vscale=vs, num_splits=splits)
        assert torch.equal(a, b)


def test_decode_out_scale_and_strided_rows():
    seg, keys = segments(21, 8, 2, [70, 5], [3, 9], False)
    q = rand(3, 2, 8, 128, gain=False).to(DEV)
    s = torch.tensor([1.5, 0.25], device=DEV)
    plain = ops.decode_attention(q, num_splits=2, **seg)
    wide = torch.zeros(2, 24, 128, dtype=BF16, device=DEV)
    wide[:, 8:16] = q
    out = torch.full((2, 16, 128), 7.0, dtype=BF16, device=DEV)
    got = ops.decode_attention(wide[:, 8:16], num_splits=2, out_scale=s, out=out[:, 4:12], **seg)
    assert torch.equal(got, (plain.float() * s.repeat_interleave(4)[:, None]).to(BF16))
    assert bool((out[:, :4] == 7).all()) and bool((out[:, 12:] == 7).all())


def test_decode_ignores_what_lies_past_a_sequence_and_keeps_nan_blocks():
    """Codes past the length may be anything; a NaN block that is seen makes its rows NaN, one that is not does nothing."""

    pool, table, k, v = history(31, 2, 2, 96, shuffle=False)
    q = rand(3, 2, 4, 128, gain=False).to(DEV)
    kw = dict(older=pool, older_table=table, older_len=torch.tensor([40, 96], dtype=torch.int32, device=DEV))
    want = ops.decode_attention(q, num_splits=1, **kw)
    u = lambda t: t.view(torch.uint8)
    src = paged(k.transpose(1, 2), v.transpose(1, 2), table)
    for t in (pool.k, pool.v):  # sequence 0's page 1: NaN codes in tokens 8 on, page 2 all NaN
        cut = ops.PagedKV8.zeros(pool.pages, 2, DEV)
        ops.kv8_quantize(src, cut, src_table=table[:1], dst_table=table[:1], tokens=40)
        kept = u(cut.k if t is pool.k else cut.v)[:, 1] != 0
        u(t)[:, 1] = torch.where(kept, u(t)[:, 1], 0x7f)
        u(t)[:, 2] = 0xff
    pool.k_scales[:, 2] = 255
    seen = ops.decode_attention(q, num_splits=1, **kw)
    assert torch.equal(seen[1], want[1])
    zero = (k[0, :, 32:40] == 0) | (v[0, :, 32:40] == 0)
    if not bool(zero.any()):
        assert torch.equal(seen[0], want[0])
    pool.v_scales[1, 4] = 255  # sequence 1's block 1 of head 1
    for splits in (1, 2, 3):
        got = ops.decode_attention(q, num_splits=splits, **kw)
        assert bool(got[1, 2:].isnan().all()) and not bool(got[1, :2].isnan().any()) and not bool(got[0].isnan().any())


@pytest.mark.parametrize("Hq,Hkv,L,older,local,vscale", [
    (8, 2, 3, [0, 33, 200], [3, 9, 50], True),        # 12 columns a kv head
    (8, 2, 7, [64, 500], [7, 40], False),             # 28
    (16, 2, 8, [64, 31], [8, 33], True),              # 64
    (8, 2, 40, [0, 100, 260], [40, 41, 90], True),    # tiles
    (4, 4, 100, [129, 700], [100, 120], False),
])
def test_prefill_against_64_bits_and_the_bf16_call(Hq, Hkv, L, older, local, vscale):
    seg, keys = segments(41, Hq, Hkv, older, local, vscale)
    B = len(older)
    q = rand(43, B, L, Hq, 128, gain=False)
    out = ops.prefill_attention(q.to(DEV), causal=True, **seg)
    for b, (k, v) in enumerate(keys):
        want, mean, err, _ = attention64(q[b], k, v, L)
        check(out[b], want, mean, err, 2.0 ** -10, b)  # (tiles carry a weight in fp16: 2^-11, and the sum's)
    k8, v8 = ops.kv8_unpack(seg["older"], seg["older_table"], 0, 32 * seg["older_table"].shape[1])
    twin = dict(seg, older=paged(k8.transpose(1, 2), v8.transpose(1, 2), seg["older_table"]))
    if L * Hq // Hkv > 64:
        assert torch.equal(out, ops.prefill_attention(q.to(DEV), causal=True, **twin))


def test_prefill_bidirectional_without_a_ring_and_fixed_lengths():
    pool, table, k, v = history(51, 2, 2, 333)
    for L in (4, 50):
        q = rand(52, 2, L, 8, 128, gain=False)
        for n in (333, 320, 1):
            out = ops.prefill_attention(q.to(DEV), causal=False, older=pool, older_table=table, older_len=n)
            for b in range(2):
                want, mean, err, _ = attention64(q[b], k[b, :, :n].cpu(), v[b, :, :n].cpu(), 0)
                check(out[b], want, mean, err, 2.0 ** -10, (L, n, b))


@pytest.mark.parametrize("splits", [0, 3])
@pytest.mark.parametrize("host", [False, True])
@pytest.mark.parametrize("counts", [[1, 1, 1], [1, 7, 1, 40], [20, 1, 33, 2, 16], [5]])
def test_ragged_prefill_against_64_bits(counts, host, splits):
    older = [97 * i % 400 for i in range(len(counts))]
    local = [n + 11 * i % 60 for i, n in enumerate(counts)]
    seg, keys = segments(61, 8, 2, older, local, True)
    cu = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
    q = rand(62, int(cu[-1]), 8, 128, gain=False)
    out = ops.prefill_attention(q.to(DEV), causal=True, cu_seqlens_q=torch.from_numpy(cu).to(DEV), max_seqlen_q=max(counts),
                                cu_seqlens_q_host=cu if host else None, num_splits=splits, **seg)
    for b, (k, v) in enumerate(keys):
        want, mean, err, _ = attention64(q[cu[b]:cu[b + 1]], k, v, counts[b])
        check(out[cu[b]:cu[b + 1]], want, mean, err, 2.0 ** -10, (b, host))


def test_large_v_takes_the_wide_tiles():
    """V beyond fp16's range in the history, through the tile kernel's bf16 instance."""

    k, v = rand(71, 1, 64, 1, 128), rand(72, 1, 64, 1, 128) * 3e5
    table = table_of(1, 2)
    pool = ops.PagedKV8.zeros(2, 1, DEV)
    ops.kv8_quantize(paged(k, v, table), pool, src_table=table, dst_table=table, tokens=64)
    k8, v8 = ops.kv8_unpack(pool, table, 0, 64)
    q = rand(73, 1, 70, 2, 128, gain=False)
    out = ops.prefill_attention(q.to(DEV), causal=False, older=pool, older_table=table, older_len=64)
    want, mean, err, _ = attention64(q[0], k8[0].cpu(), v8[0].cpu(), 0)
    check(out[0], want, mean, err, 2.0 ** -10)


def test_captured_decode_and_prefill_replay():
    """One graph of both calls, replayed with other inputs and eager work between."""

    seg, keys = segments(81, 8, 2, [300, 77], [40, 41], True)
    q1, qL = rand(82, 2, 8, 128, gain=False).to(DEV), rand(83, 2, 40, 8, 128, gain=False).to(DEV)
    ws1 = torch.empty(ops.decode_workspace_bytes(2, 8, 4), dtype=torch.uint8, device=DEV)
    ws2 = torch.empty(ops.prefill_kv8_workspace_bytes(2, 2, 32 * seg["older_table"].shape[1], 128, query_rows=80, num_q_heads=8),
                      dtype=torch.uint8, device=DEV)
    o1, oL = torch.empty_like(q1), torch.empty_like(qL)

    def both():
        ops.decode_attention(q1, num_splits=4, workspace=ws1, out=o1, **seg)
        ops.prefill_attention(qL, causal=True, workspace=ws2, out=oL, **seg)

    both()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        both()
    for i in range(4):
        q1.copy_(rand(90 + i, 2, 8, 128, gain=False))
        qL.copy_(rand(95 + i, 2, 40, 8, 128, gain=False))
        o1.zero_()
        oL.zero_()
        g.replay()
        torch.cuda.synchronize()
        a, b = o1.clone(), oL.clone()
        both()
        torch.cuda.synchronize()
        assert torch.equal(a, o1) and torch.equal(b, oL)


def test_runs_on_the_current_stream():
    k, v = rand(3, 1, 64, 2, 128).to(DEV), rand(4, 1, 64, 2, 128).to(DEV)
    table = table_of(1, 2)
    src = paged(k, v, table)
    pool, again = ops.PagedKV8.zeros(2, 2, DEV), ops.PagedKV8.zeros(2, 2, DEV)
    ops.kv8_quantize(src, again, src_table=table, dst_table=table, tokens=64)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        torch.cuda._sleep(20_000_000)
        ops.kv8_quantize(src, pool, src_table=table, dst_table=table, tokens=64)
        got = ops.kv8_unpack(pool, table, 0, 64)
    s.synchronize()
    want = ops.kv8_unpack(again, table, 0, 64)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


# ---------------------------------------------------------------------------------------- refusals
def test_refusals():
    pool, table, k, v = history(91, 2, 2, 64)
    bf = paged(k.transpose(1, 2), v.transpose(1, 2), table)
    q = rand(1, 2, 4, 128).to(DEV)
    err = (ValueError, ops._lib.LastKVNativeError)
    for kw in (dict(older=pool, older_len=3), dict(older=pool, older_table=table.long(), older_len=3),
               dict(older=pool, older_table=table, older_len=65), dict(older=pool, older_table=table[:1], older_len=3),
               dict(older=pool, older_table=table, older_len=3, older_slot=table[:, 0].contiguous()),
               dict(older=bf, older_table=table, older_len=3, local=pool, local_table=table, local_len=1),
               dict(older=pool, older_table=table, older_len=3, no_alloc=True)):
        with pytest.raises(err):
            ops.decode_attention(q, **kw)
    with pytest.raises(err):
        ops.prefill_attention(q[:, None].expand(2, 40, 4, 128).contiguous(), older=pool, older_table=table, older_len=64,
                              workspace=torch.empty(1024, dtype=torch.uint8, device=DEV))
    ok = dict(src_table=table, dst_table=table, tokens=64)
    for args, kw in (((bf, bf), ok), ((pool, pool), ok), ((bf, ops.PagedKV8.zeros(4, 3, DEV)), ok),
                     ((bf, pool), dict(ok, tokens=-1)), ((bf, pool), dict(ok, tokens=None)), ((bf, pool), dict(ok, blocks=3)),
                     ((bf, pool), dict(ok, first_block=-1)), ((bf, pool), dict(ok, dst_table=table[:1])),
                     ((bf, pool), dict(ok, src_table=table.float())), ((bf, pool), dict(ok, tokens=torch.zeros(2, device=DEV)))):
        with pytest.raises(err):
            ops.kv8_quantize(*args, **kw)
    for a in ((bf, table, 0, 4), (pool, table, 0, 65), (pool, table, -1, 4), (pool, table[0], 0, 4)):
        with pytest.raises(err):
            ops.kv8_unpack(*a)
    with pytest.raises(err):
        ops.PagedKV8(pool.k, pool.v, pool.k_scales[:, :1], pool.v_scales)
    with pytest.raises(err):
        ops.PagedKV8(pool.k.view(torch.uint8), pool.v, pool.k_scales, pool.v_scales)
