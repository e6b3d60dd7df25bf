"""The 8-bit cache's operators, page copies and beam selection as they are called: the native launch path against the Python
bodies, the torch custom operators, copy-on-write outputs, errors, empty batches, and offsets past 32 bits (gpu)."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import lastkv_amd.torch_ops  # noqa: F401
from lastkv_amd import _lib, ops
import test_gpu_search as search
from test_gpu_host_path import _both
from test_gpu_kv8 import DEV, attention64, check, history, paged, rand, segments, table_of

pytestmark = pytest.mark.gpu
L = torch.ops.lastkv
FLOAT8 = ("test_faketensor", "test_autograd_registration")  # (the other checks multiply their inputs, which float8 has not)


def i32(*x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def four(p):
    return p.k, p.v, p.k_scales, p.v_scales


# ---------------------------------------------------------------------------------------- one call, two ways
@pytest.mark.parametrize("call", ["plain", "strided4d", "outputs", "splits", "scale", "alone"])
def test_decode_native_and_python(call, monkeypatch):
    seg, _ = segments(3, 8, 2, [70, 0, 33], [5, 40, 0], True)
    if call == "alone":
        seg = {k: v for k, v in seg.items() if not k.startswith("local")}
    q = rand(4, 3, 3 * 8, 128).to(DEV)[:, 8:16] if call == "strided4d" else rand(4, 3, 8, 128).to(DEV)

    def make():
        kw = dict(seg)
        if call == "outputs":
            kw.update(out=torch.zeros(3, 8, 128, dtype=torch.bfloat16, device=DEV), lse=torch.zeros(3, 8, device=DEV),
                      workspace=torch.empty(1 << 20, dtype=torch.uint8, device=DEV))
        if call == "splits":
            kw.update(num_splits=2, sm_scale=0.05)
        if call == "scale":
            kw.update(out_scale=torch.full((2,), 0.75, device=DEV), vscale=None)
        out = ops.decode_attention(q, **kw)
        return (out, kw["lse"]) if call == "outputs" else (out,)

    _both(monkeypatch, make)


@pytest.mark.parametrize("B", [32, 34, 40, 64])
def test_default_splits_of_many_sequences(B, monkeypatch):
    """More (sequence, kv head) pairs than CUs: both ways choose the splits that ``default_decode_splits`` names."""

    pool, table, _, _ = history(28, 1, 8, 4200)
    rows = table.expand(B, -1).contiguous()
    q = rand(29, B, 8, 128).to(DEV)
    splits = ops.default_decode_splits(B, 8, 4200, ops._cu_count(q.device), True)
    call = lambda **kw: (ops.decode_attention(q, older=pool, older_table=rows, older_len=4200, **kw),)
    _both(monkeypatch, call)
    assert torch.equal(call()[0], call(num_splits=splits)[0])


@pytest.mark.parametrize("call", ["plain", "ragged", "ragged_host", "both"])
@pytest.mark.parametrize("tokens", [3, 40])
def test_prefill_native_and_python(call, tokens, monkeypatch):
    local = [tokens, tokens + 7, tokens]
    seg, _ = segments(5, 8, 2, [70, 0, 33], local, False)
    lens = [tokens, 1, 0] if "ragged" in call else None
    q = rand(6, *((sum(lens),) if lens else (3, tokens)), 8, 128).to(DEV)
    cu = np.concatenate(([0], np.cumsum(lens))).astype(np.int32) if lens else None

    def make():
        kw = dict(seg, lse=torch.zeros(q.shape[:-1], device=DEV))
        if lens:
            kw.update(cu_seqlens_q=torch.from_numpy(cu).to(DEV), max_seqlen_q=tokens)
        if call == "ragged_host":
            kw.update(cu_seqlens_q_host=cu)
        if call == "both":
            kw.update(causal=False)
        return ops.prefill_attention(q, **kw), kw["lse"]

    _both(monkeypatch, make)


def test_other_calls_native_and_python(monkeypatch):
    pool, table, k, v = history(7, 2, 2, 96)
    src = paged(k.transpose(1, 2), v.transpose(1, 2), table)

    def quantize(tokens, **kw):
        def make():
            dst = ops.PagedKV8.zeros(7, 2, DEV)
            ops.kv8_quantize(src, dst, src_table=table, dst_table=table, tokens=tokens, **kw)
            return four(dst)[:2] + four(dst)[2:]
        return lambda: tuple(t.view(torch.uint8) for t in make())

    _both(monkeypatch, quantize(96))
    _both(monkeypatch, quantize(i32(96, 40), first_block=1, blocks=2))
    _both(monkeypatch, lambda: ops.kv8_unpack(pool, table, 3, 50))

    def copy(first, second):
        def make():
            p = ops.PagedKV8(*(t.clone() for t in four(pool)))
            ops.copy_pages(p, first, second)
            return tuple(t.view(torch.uint8) for t in four(p))
        return make

    _both(monkeypatch, copy(np.array([0, 1], dtype=np.int32), np.array([4, 5], dtype=np.int32)))
    _both(monkeypatch, copy([0, 1], [4, 5]), native=False)  # (what is no int32 array goes the Python way)
    _both(monkeypatch, copy(np.array([0], dtype=np.int64), np.array([2], dtype=np.int32)), native=False)
    for dtype in (torch.bfloat16, torch.float32):
        logits = torch.randn(2, 3, 999, device=DEV).to(dtype)
        scores = -torch.rand(2, 3, device=DEV)
        _both(monkeypatch, lambda: ops.beam_select(logits, scores, 6))
        ws = torch.empty(ops.beam_workspace_bytes(2, 3, 999, 6), dtype=torch.uint8, device=DEV)
        _both(monkeypatch, lambda: ops.beam_select(logits, scores, 6, workspace=ws))


# ---------------------------------------------------------------------------------------- torch custom operators
def test_custom_operators():
    seg, _ = segments(8, 8, 2, [70, 0, 33], [45, 40, 41], True)
    pool, ring = seg["older"], seg["local"]
    rest = (seg["older_len"], 0, seg["older_table"], seg["vscale"], ring.k, ring.v, seg["local_len"], 0,
            seg["local_start"], 0, seg["local_table"], 4)
    q = rand(9, 3, 8, 128).to(DEV)
    args = (q, *four(pool), *rest, 0.0, 0)
    assert torch.equal(L.decode_attention_kv8(*args), ops.decode_attention(q, **seg))
    torch.library.opcheck(L.decode_attention_kv8, args, test_utils=FLOAT8)
    qp = rand(10, 3, 40, 8, 128).to(DEV)
    args = (qp, *four(pool), *rest, True, 0.0)
    assert torch.equal(L.prefill_attention_kv8(*args), ops.prefill_attention(qp, **seg))
    torch.library.opcheck(L.prefill_attention_kv8, args, test_utils=FLOAT8)
    cu = i32(0, 40, 41, 48)
    args = (qp.view(-1, 8, 128)[:48], *four(pool), *rest, True, 0.0, None, cu, 40, 0, cu.cpu())
    assert torch.equal(L.prefill_attention_kv8(*args), ops.prefill_attention(
        args[0], cu_seqlens_q=cu, max_seqlen_q=40, cu_seqlens_q_host=cu.cpu().numpy(), **seg))
    torch.library.opcheck(L.prefill_attention_kv8, args, test_utils=FLOAT8)

    table = seg["older_table"]
    assert all(torch.equal(a, b) for a, b in zip(L.kv8_unpack(*four(pool), table, 3, 20), ops.kv8_unpack(pool, table, 3, 20)))
    torch.library.opcheck(L.kv8_unpack, (*four(pool), table, 3, 20), test_utils=FLOAT8)
    src = ops.PagedKV(*(rand(s, 2, pool.pages, 4096).to(DEV) for s in (11, 12)))
    a, b = (ops.PagedKV8.zeros(pool.pages, 2, DEV) for _ in range(2))
    L.kv8_quantize(src.k, src.v, *four(a), table, table, None, 60)
    ops.kv8_quantize(src, b, src_table=table, dst_table=table, tokens=60)
    assert all(torch.equal(x.view(torch.uint8), y.view(torch.uint8)) for x, y in zip(four(a), four(b)))
    torch.library.opcheck(L.kv8_quantize, (src.k, src.v, *four(a), table, table, seg["older_len"], 0, 0, 1), test_utils=FLOAT8)
    L.copy_pages(*four(a), [0, 1], [2, 4])
    ops.copy_pages(b, [0, 1], [2, 4])
    assert all(torch.equal(x.view(torch.uint8), y.view(torch.uint8)) for x, y in zip(four(a), four(b)))
    torch.library.opcheck(L.copy_pages, (src.k, src.v, None, None, [0, 1], [2, 4]))
    logits, scores = torch.randn(2, 3, 700, device=DEV), -torch.rand(2, 3, device=DEV)
    assert all(torch.equal(x, y) for x, y in zip(L.beam_select(logits, scores, 6), ops.beam_select(logits, scores, 6)))
    torch.library.opcheck(L.beam_select, (logits, scores, 6))


def test_a_compiled_fragment_equals_eager():
    pool, table, _, _ = history(13, 2, 2, 100)
    wq = rand(14, 1024, 1024).to(DEV) * 0.02
    head = rand(15, 1024, 500).to(DEV) * 0.02

    def step(h, scores):
        o = L.decode_attention_kv8((h @ wq).view(2, 8, 128), *four(pool), None, 100, table, None, None, None, None, 0, None, 0,
                                   None, 0, 0.0, 0)
        return L.beam_select((o.reshape(1, 2, 1024) @ head), scores, 4)

    h, scores = rand(16, 2, 1024).to(DEV), torch.zeros(1, 2, device=DEV)
    for a, b in zip(torch.compile(step, backend="aot_eager", fullgraph=True)(h, scores), step(h, scores)):
        assert torch.equal(a, b)


# ---------------------------------------------------------------------------------------- outputs, errors, empty calls
def test_written_tensors_detach_copy_on_write():
    pool, table, k, v = history(17, 1, 2, 64)
    src = paged(k.transpose(1, 2), v.transpose(1, 2), table)
    kept = []

    def lazy(t):
        kept.append((t, t.clone(), torch._lazy_clone(t)))
        return kept[-1][2]

    dst = ops.PagedKV8(*(lazy(t) for t in four(ops.PagedKV8.zeros(2, 2, DEV))))
    ops.kv8_quantize(src, dst, src_table=table, dst_table=table, tokens=64)
    copied = ops.PagedKV(lazy(src.k), lazy(src.v))
    ops.copy_pages(copied, *(np.array([i], dtype=np.int32) for i in (0, 1)))
    q = rand(18, 1, 4, 128).to(DEV)
    ops.decode_attention(q, older=pool, older_table=table, older_len=64, num_splits=2, out=lazy(torch.zeros_like(q)),
                         lse=lazy(torch.zeros(1, 4, device=DEV)), workspace=lazy(torch.zeros(1 << 18, dtype=torch.uint8, device=DEV)))
    ws = lazy(torch.zeros(ops.beam_workspace_bytes(1, 2, 500, 4), dtype=torch.uint8, device=DEV))
    ops.beam_select(torch.randn(1, 2, 500, device=DEV), torch.zeros(1, 2, device=DEV), 4, workspace=ws)
    torch.cuda.synchronize()
    for original, before, written in kept:
        as_bytes = [t.view(torch.uint8) for t in (original, before, written)]
        assert torch.equal(as_bytes[0], as_bytes[1]) and not torch.equal(as_bytes[0], as_bytes[2])


@pytest.mark.parametrize("op", ["decode", "prefill", "quantize", "unpack", "copy", "beam"])
def test_a_reported_hip_error_raises(op):
    pool, table, k, v = history(19, 1, 2, 64)
    src = paged(k.transpose(1, 2), v.transpose(1, 2), table)
    q = rand(20, 1, 4, 128).to(DEV)
    seg = dict(older=pool, older_table=table, older_len=64)
    logits, scores = torch.randn(1, 2, 500, device=DEV), torch.zeros(1, 2, device=DEV)
    calls = {
        "decode": lambda: ops.decode_attention(q, num_splits=1, **seg),
        "prefill": lambda: ops.prefill_attention(q[:, None], **seg),
        "quantize": lambda: ops.kv8_quantize(src, pool, src_table=table, dst_table=table, tokens=64),
        "unpack": lambda: ops.kv8_unpack(pool, table, 0, 64),
        "copy": lambda: ops.copy_pages(src, [0], [1]),
        "beam": lambda: ops.beam_select(logits, scores, 4),
    }
    calls[op]()
    torch.cuda.synchronize()
    assert _lib.load().hipSetDevice(9999) != 0  # (resolved from the HIP runtime the library is linked with)
    with pytest.raises(_lib.LastKVNativeError, match="status 4"):
        calls[op]()
    torch.cuda.synchronize()


def test_empty_calls():
    pool, table, k, v = history(21, 2, 2, 64)
    src = paged(k.transpose(1, 2), v.transpose(1, 2), table)
    before = [t.clone() for t in four(pool)]
    none = table[:0]
    q = rand(22, 2, 4, 128).to(DEV)
    ops.kv8_quantize(src, pool, src_table=none, dst_table=none, tokens=64)
    ops.kv8_quantize(src, pool, src_table=table, dst_table=table, tokens=0)
    ops.kv8_quantize(src, pool, src_table=table, dst_table=table, tokens=64, blocks=0)
    ops.copy_pages(pool, [], [])
    assert ops.kv8_unpack(pool, table, 5, 0)[0].shape == (2, 2, 0, 128)
    assert ops.kv8_unpack(pool, none, 0, 5)[1].shape == (0, 2, 5, 128)
    assert [t.shape for t in ops.beam_select(torch.zeros(0, 2, 9, device=DEV), torch.zeros(0, 2, device=DEV), 3)] == [(0, 3)] * 3
    # a history of no tokens and no ring: no key at all, so zeros with an LSE of -inf
    lse = torch.zeros(2, 4, device=DEV)
    assert not ops.decode_attention(q, older=pool, older_table=table, older_len=0, lse=lse).any()
    assert bool((lse == -torch.inf).all())
    torch.cuda.synchronize()
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(before, four(pool)))


# ---------------------------------------------------------------------------------------- large pools
def test_offsets_past_32_bits():
    """A pool whose later heads' and pages' bytes lie past 2^32 (2 x 600000 x 4096 of codes each): quantised, read back, and
    attended to by single tokens and by rows of queries."""

    pages, H, T = 600000, 2, 100
    pool = ops.PagedKV8(*(torch.empty((H, pages, 4096), dtype=torch.float8_e4m3fn, device=DEV) for _ in range(2)),
                        *(torch.zeros((H, pages), dtype=torch.uint8, device=DEV) for _ in range(2)))
    try:
        table = i32(*range(pages - 4, pages)).view(1, 4)
        k, v = rand(23, 1, 128, H, 128), rand(24, 1, 128, H, 128)
        small = table_of(1, 4)
        src = paged(k, v, small)
        ops.kv8_quantize(src, pool, src_table=small, dst_table=table, tokens=T)
        near = ops.PagedKV8.zeros(4, H, DEV)
        ops.kv8_quantize(src, near, src_table=small, dst_table=small, tokens=T)
        for a, b in zip(ops.kv8_unpack(pool, table, 0, T), ops.kv8_unpack(near, small, 0, T)):
            assert torch.equal(a, b)
        q = rand(25, 1, 40, 8, 128).to(DEV)
        for call in (lambda p, t: ops.decode_attention(q[:, 0].contiguous(), older=p, older_table=t, older_len=T),
                     lambda p, t: ops.prefill_attention(q, older=p, older_table=t, older_len=T),
                     lambda p, t: ops.prefill_attention(q[:, :3].contiguous(), older=p, older_table=t, older_len=T)):
            assert torch.equal(call(pool, table), call(near, small))
        ops.copy_pages(pool, [pages - 4, pages - 1], [5, 4])
        assert torch.equal(pool.k[:, 5].view(torch.uint8), pool.k[:, pages - 4].view(torch.uint8))
        assert torch.equal(pool.v_scales[:, 4], pool.v_scales[:, pages - 1])
    finally:
        del pool
        torch.cuda.empty_cache()


@pytest.mark.parametrize("splits", [None, 1, 4, 7, 64])
@pytest.mark.parametrize("older", [[8192, 8191], [8193, 255 * 32], [12345, 33], [32768, 32 * 1024 - 31], [34000, 32 * 1023]])
def test_long_decode_rows(older, splits):
    """Histories of 255 blocks and more, which the splits of a call begin to read at different places."""

    seg, keys = segments(30, 8, 2, older, [9, 64], True)
    q = rand(31, 2, 8, 128).to(DEV)
    got = ops.decode_attention(q, num_splits=splits, **seg)
    for b in range(2):
        want, mean, err, _ = attention64(q[b:b + 1].cpu(), *keys[b], 0)
        check(got[b:b + 1], want, mean, err, 2.0 ** -8, b)  # (weights rounded to bf16: 2^-8 at most)


@pytest.mark.parametrize("T", [4000, 9001])
def test_long_ragged_batches(T):
    """Ragged rows over long histories: a prompt's chunk, a few tokens, one token, and none."""

    counts = [130, 5, 1, 0]
    seg, keys = segments(26, 8, 2, [T, 33, T - 1, 64], [130, 5, 1, 7], True, ring_blocks=5)
    q = rand(27, sum(counts), 8, 128).to(DEV)
    cu = np.concatenate(([0], np.cumsum(counts))).astype(np.int32)
    for kw in ({}, dict(cu_seqlens_q_host=cu)):
        got = ops.prefill_attention(q, cu_seqlens_q=torch.from_numpy(cu).to(DEV), max_seqlen_q=130, **kw, **seg)
        for b, n in enumerate(counts):
            if n:
                rows = slice(int(cu[b]), int(cu[b + 1]))
                want, mean, err, _ = attention64(q[rows].cpu(), *keys[b], n)
                # weights rounded to bf16 (2^-8 at most) or V to fp16 (2^-11): the larger
                check(got[rows], want, mean, err, 2.0 ** -8, (T, b))


# ---------------------------------------------------------------------------------------- calls at their edges
@pytest.mark.parametrize("host", [False, True])
@pytest.mark.parametrize("counts", [[3, 1], [70, 1, 9], [1, 1]])
def test_rows_behind_the_last_sequence_stay(counts, host):
    """A padded ragged batch: rows past the last offset are neither read nor written, nor are their LSEs."""

    seg, _ = segments(32, 8, 2, [200, 64, 33][:len(counts)], [n + 5 for n in counts], True)
    T = sum(counts)
    q = rand(33, T + 11, 8, 128).to(DEV)
    cu = np.concatenate(([0], np.cumsum(counts))).astype(np.int32)
    kw = dict(cu_seqlens_q=torch.from_numpy(cu).to(DEV), max_seqlen_q=max(counts), **(dict(cu_seqlens_q_host=cu) if host else {}), **seg)
    want = ops.prefill_attention(q[:T].contiguous(), **kw)
    out, lse = torch.full_like(q, 7.0), torch.full((T + 11, 8), 7.0, device=DEV)
    q[T:] = float("nan")
    ops.prefill_attention(q, out=out, lse=lse, **kw)
    assert torch.equal(out[:T], want) and bool((out[T:] == 7).all()) and bool((lse[T:] == 7).all())


def test_table_entries_past_a_length_are_not_followed():
    pool, table, _, _ = history(34, 2, 2, 300)
    wide = torch.full((2, 40), -5, dtype=torch.int32, device=DEV)
    wide[:, ::2] = 1 << 30
    wide[:, :10] = table
    q = rand(35, 2, 40, 8, 128).to(DEV)
    lens = i32(300, 33)
    for n in (1, 3, 40):
        rows = q[:, :n].contiguous()
        a, b = (ops.prefill_attention(rows, older=pool, older_table=t, older_len=lens, num_splits=1) for t in (table, wide))
        assert torch.equal(a, b)
    a, b = (ops.decode_attention(q[:, 0].contiguous(), older=pool, older_table=t, older_len=lens, num_splits=3) for t in (table, wide))
    assert torch.equal(a, b)


@pytest.mark.parametrize("T", [0, 1, 31, 32])
def test_shortest_histories(T):
    seg, keys = segments(36, 16, 1, [T, 0], [1, 1], True)
    for L in (1, 2, 5):
        q = rand(37, 2, L, 16, 128).to(DEV)
        local = [L, L]
        seg, keys = segments(36, 16, 1, [T, 0], local, True)
        got = ops.prefill_attention(q, **seg) if L > 1 else ops.decode_attention(q[:, 0].contiguous(), **seg)[:, None]
        for b in range(2):
            want, mean, err, _ = attention64(q[b].cpu(), *keys[b], L)
            check(got[b], want, mean, err, 2.0 ** -8, (T, L, b))  # (weights rounded to bf16: 2^-8 at most)


def test_strided_logits_and_scores():
    """Views of larger tensors, against 64 bits (which values a thread adds up in fp32 goes by a row's alignment, so a copy's
    scores may differ in their last bit)."""

    g = torch.Generator(device=DEV).manual_seed(39)
    logits = torch.randn((4, 6, 3000), generator=g, device=DEV)[::2, 1::2, 7:2900]
    scores = -torch.rand((4, 9), generator=g, device=DEV)[::2, 3:6]
    search.check(logits, scores, 6)
    for bad in (torch.randn(2, 3000, 3, device=DEV).transpose(1, 2), logits.double(), logits[0], logits.cpu()):
        with pytest.raises((ValueError, _lib.LastKVNativeError)):
            ops.beam_select(bad, scores, 6)


def test_calls_on_two_streams():
    """Two calls in flight at once, each with its own workspace, give what they give alone."""

    segs = [segments(38 + i, 8, 2, [5000 + i, 77], [9, 30], True)[0] for i in range(2)]
    qs = [rand(40 + i, 2, 8, 128).to(DEV) for i in range(2)]
    logits = [torch.randn(2, 4, 50000, device=DEV) for _ in range(2)]
    scores = torch.zeros(2, 4, device=DEV)
    alone = [(ops.decode_attention(q, num_splits=8, **s), *ops.beam_select(x, scores, 8)) for q, s, x in zip(qs, segs, logits)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(3):
        got = []
        for st, q, s, x in zip(streams, qs, segs, logits):
            with torch.cuda.stream(st):
                got.append((ops.decode_attention(q, num_splits=8, **s), *ops.beam_select(x, scores, 8)))
        torch.cuda.synchronize()
        for a, b in zip(alone, got):
            assert all(torch.equal(x, y) for x, y in zip(a, b))
