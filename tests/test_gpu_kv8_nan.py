"""NaN blocks of an 8-bit history, values past a length, and the LSE of calls of several query tokens (gpu)."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from lastkv_amd import ops
from test_gpu_kv8 import DEV, attention64, history, rand, segments

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
