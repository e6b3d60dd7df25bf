"""NaN blocks of an 8-bit history, values past a length, and the LSE of calls of several query tokens (gpu)."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from lastkv_amd import ops
from test_gpu_kv8 import DEV, attention64, history, paged, rand, segments, table_of

pytestmark = pytest.mark.gpu


def i32(*x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


CALLS = {  # query tokens of each sequence (32 or 8 query heads over 2 kv heads), arguments, whether the call is ragged
    "decode": (1, 8, dict(num_splits=1), False),
    "decode_splits": (1, 8, dict(num_splits=3), False),
    "wide_group": (1, 64, dict(num_splits=2), False),
    "short": (3, 8, dict(), False),
    "short_splits": (7, 8, dict(num_splits=3), False),
    "tiles": (40, 8, dict(num_splits=1), False),
    "tiles8": (40, 8, dict(num_splits=1, tile_waves=8), False),
    "halves": (40, 8, dict(), False),
    "narrow_tiles": (9, 8, dict(tile_waves=4), False),
    "ragged": (40, 8, dict(num_splits=1), True),
    "ragged_splits": (40, 8, dict(), True),
    "ragged_short": (5, 8, dict(), True),
}


def attend(name, q, lse, **kw):
    tokens, _, extra, ragged = CALLS[name]
    if name.startswith(("decode", "wide")):
        return ops.decode_attention(q[:, 0].contiguous(), lse=lse[:, 0], **extra, **kw)[:, None]
    if not ragged:
        return ops.prefill_attention(q, causal=False, lse=lse, **extra, **kw)
    B = q.shape[0]
    cu = np.arange(0, B * tokens + 1, tokens, dtype=np.int32)
    return ops.prefill_attention(q.flatten(0, 1), causal=False, lse=lse.flatten(0, 1), cu_seqlens_q=torch.from_numpy(cu).to(DEV),
                                 max_seqlen_q=tokens, cu_seqlens_q_host=cu, **extra, **kw).view_as(q)


@pytest.mark.parametrize("which", ["k", "v", "both"])
@pytest.mark.parametrize("T,block", [(20, 0), (700, 0), (700, 9), (700, 21), (2100, 33)])
@pytest.mark.parametrize("name", CALLS)
def test_a_visible_nan_block_makes_output_and_lse_nan(name, T, block, which):
    """Of every row of its sequence and kv head, and of no other; also where the history is that block alone."""

    tokens, Hq, _, _ = CALLS[name]
    pool, table, _, _ = history(T, 2, 2, T)
    q = rand(7, 2, tokens, Hq, 128, gain=False).to(DEV)
    lens = i32(T, T)
    lse, before = (torch.zeros(2, tokens, Hq, device=DEV) for _ in range(2))
    want = attend(name, q, before, older=pool, older_table=table, older_len=lens)
    for t in ("k", "v"):
        if which in (t, "both"):
            getattr(pool, t + "_scales")[1, int(table[0, block])] = 255
    got = attend(name, q, lse, older=pool, older_table=table, older_len=lens)
    hit = torch.zeros(2, 1, Hq, dtype=torch.bool, device=DEV)
    hit[0, :, Hq // 2:] = True
    assert torch.equal(got.isnan().all(-1), hit.expand(2, tokens, Hq)) and torch.equal(got.isnan().any(-1), hit.expand(2, tokens, Hq))
    assert torch.equal(lse.isnan(), hit.expand(2, tokens, Hq)), lse[0, 0]
    keep = ~hit.expand(2, tokens, Hq)
    assert torch.equal(got[keep], want[keep]) and torch.equal(lse[keep], before[keep])


@pytest.mark.parametrize("name", CALLS)
def test_a_nan_block_past_a_length_does_nothing(name):
    tokens, Hq, _, _ = CALLS[name]
    pool, table, _, _ = history(9, 2, 2, 640)
    q = rand(7, 2, tokens, Hq, 128, gain=False).to(DEV)
    lens = i32(320, 33)
    lse, before = (torch.zeros(2, tokens, Hq, device=DEV) for _ in range(2))
    want = attend(name, q, before, older=pool, older_table=table, older_len=lens)
    pool.k_scales[:, table[0, 10].long()] = 255
    pool.v_scales[:, table[1, 2].long()] = 255
    got = attend(name, q, lse, older=pool, older_table=table, older_len=lens)
    assert torch.equal(got, want) and torch.equal(lse, before)


@pytest.mark.parametrize("name", CALLS)
@pytest.mark.parametrize("T", [1, 40, 321])
def test_codes_past_a_length_may_be_anything(name, T):
    """Every code of the last block's tokens past the length, by its place in the block, becomes NaN or the greatest value."""

    tokens, Hq, _, _ = CALLS[name]
    pool, table, _, _ = history(31, 2, 2, 384)
    q = rand(3, 2, tokens, Hq, 128, gain=False).to(DEV)
    lens = i32(T, 384)
    lse, before = (torch.zeros(2, tokens, Hq, device=DEV) for _ in range(2))
    want = attend(name, q, before, older=pool, older_table=table, older_len=lens)
    at = np.arange(4096)  # byte = piece * 1024 + lane * 16 + i
    piece, lane, i = at // 1024, at // 16 % 64, at % 16
    token_k = ((lane % 16) // 4) * 8 + (piece // 2) * 4 + lane % 4
    token_v = (lane // 16) * 8 + i % 8
    page = int(table[0, T // 32])
    for t, token in ((pool.k, token_k), (pool.v, token_v)):
        past = torch.from_numpy(token >= T % 32).to(DEV)
        bytes_ = t.view(torch.uint8)
        for code in (0x7f, 0x7e, 0xff):
            bytes_[:, page] = torch.where(past, torch.tensor(code, dtype=torch.uint8, device=DEV), bytes_[:, page])
            got = attend(name, q, lse, older=pool, older_table=table, older_len=lens)
            assert torch.equal(got, want) and torch.equal(lse, before), hex(code)


@pytest.mark.parametrize("Hq,Hkv,L,older,local,kw", [
    (8, 2, 3, [0, 33, 200], [3, 9, 50], dict()),
    (16, 2, 8, [64, 31], [8, 33], dict(num_splits=2)),
    (8, 2, 40, [0, 100, 260], [40, 41, 90], dict()),
    (8, 2, 40, [0, 100, 260], [40, 41, 90], dict(tile_waves=8)),
    (4, 4, 100, [129, 700], [100, 120], dict(num_splits=1)),
    (8, 1, 30, [2100], [40], dict()),
])
@pytest.mark.parametrize("causal", [False, True])
def test_the_lse_of_prefill_against_64_bits(Hq, Hkv, L, older, local, kw, causal):
    """A score is off by `err`, and so its sum's logarithm; a tile rounds each weight of the sum to fp16: by 2^-11 of it, or by
    2^-25 where the largest is 1."""

    seg, keys = segments(41, Hq, Hkv, older, local, True)
    q = rand(43, len(older), L, Hq, 128, gain=False)
    lse = torch.zeros(len(older), L, Hq, device=DEV)
    ops.prefill_attention(q.to(DEV), causal=causal, lse=lse, **kw, **seg)
    for b, (k, v) in enumerate(keys):
        _, _, err, want = attention64(q[b], k, v, L if causal else 0)
        off = (lse[b].double().cpu() - want).abs()
        room = err + 2.0 ** -11 + k.shape[1] * 2.0 ** -25 + 2.0 ** -20 * (1 + float(want.abs().max()))
        assert float(off.max()) <= room, (b, float(off.max()), room)


@pytest.mark.parametrize("name", CALLS)
def test_zeros_beside_a_large_value_stay_zeros_under_a_scale(name):
    """V is bf16(value * vscale): where a block's power of two times vscale lies beyond fp32, the zeros of the block are 0 all the
    same, and so are the outputs that only zeros go into."""

    tokens, Hq, _, _ = CALLS[name]
    k, v = rand(1, 1, 64, 2, 128), torch.zeros(1, 64, 2, 128).bfloat16()
    v[0, 3, :, 5] = 3e38
    v[0, 40:, :, 7] = 0.25
    table = table_of(1, 2)
    pool = ops.PagedKV8.zeros(2, 2, DEV)
    ops.kv8_quantize(paged(k, v, table), pool, src_table=table, dst_table=table, tokens=64)
    q = rand(2, 1, tokens, Hq, 128, gain=False).to(DEV)
    lse = torch.zeros(1, tokens, Hq, device=DEV)
    out = attend(name, q, lse, older=pool, older_table=table, older_len=i32(64), vscale=torch.tensor([512.0, 1024.0], device=DEV))
    # (dim 5 holds an infinity, whose product with a weight's second, smaller half may be a NaN)
    assert not bool(out[..., 5].isfinite().any()) and bool(out[..., 7].isfinite().all()) and bool((out[..., 7] > 0).all())
    rest = [d for d in range(128) if d not in (5, 7)]
    assert bool((out[..., rest] == 0).all())


@pytest.mark.parametrize("factor,scales", [(2.0 ** -126, [2.0 ** 100, 1.375 * 2.0 ** 110]), (2.0 ** 118, [2.0 ** -100, 1.375 * 2.0 ** -115]),
                                           (2.0 ** -10, [-0.8203125, 1.5])])
@pytest.mark.parametrize("Hq,splits", [(8, 1), (8, 2), (64, 1)])
def test_scaled_values_of_any_magnitude_are_the_bf16_calls(Hq, splits, factor, scales):
    """Down to bf16's subnormal values and up to its largest: a block a wave, equal to the call over the same values in every bit."""

    table = table_of(2, 4)
    k = rand(5, 2, 128, 2, 128)
    v = (rand(6, 2, 128, 2, 128).float() * factor).bfloat16()
    pool = ops.PagedKV8.zeros(8, 2, DEV)
    ops.kv8_quantize(paged(k, v, table), pool, src_table=table, dst_table=table, tokens=128)
    k8, v8 = ops.kv8_unpack(pool, table, 0, 128)
    twin = paged(k8.transpose(1, 2), v8.transpose(1, 2), table)
    q = rand(7, 2, Hq, 128, gain=False).to(DEV)
    kw = dict(older_table=table, older_len=i32(100, 128), vscale=torch.tensor(scales, device=DEV), num_splits=splits)
    assert torch.equal(ops.decode_attention(q, older=pool, **kw), ops.decode_attention(q, older=twin, **kw))
