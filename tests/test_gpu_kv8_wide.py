"""Prefill over 8-bit pages whose V lies beyond fp16: the tiles that read it from the codes (gpu)."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from lastkv_amd import ops
from test_gpu_kv8 import DEV, paged, rand, table_of

pytestmark = pytest.mark.gpu


def i32(*x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def pools(seed, B, H, T, large):
    """An 8-bit pool and its bf16 twin; `large`: (sequence, head, token) triples whose V is beyond fp16."""

    table = table_of(B, T // 32, seed)
    k, v = rand(seed, B, T, H, 128), rand(seed + 1, B, T, H, 128)
    for b, h, t in large:
        v[b, t, h] *= 3e5
    pool = ops.PagedKV8.zeros(table.numel(), H, DEV)
    ops.kv8_quantize(paged(k, v, table), pool, src_table=table, dst_table=table, tokens=T)
    k8, v8 = ops.kv8_unpack(pool, table, 0, T)
    return pool, paged(k8.transpose(1, 2), v8.transpose(1, 2), table), table


@pytest.mark.parametrize("ring", ["none", "paged", "tiled"])
@pytest.mark.parametrize("vscale", [False, True])
@pytest.mark.parametrize("L,G,kw", [(40, 2, dict()), (40, 4, dict(tile_waves=4)), (300, 4, dict(tile_waves=8)), (9, 4, dict(tile_waves=4)),
                                    (40, 2, dict(num_splits=1)), (17, 4, dict())])
def test_wide_tiles_equal_the_bf16_calls(L, G, kw, vscale, ring):
    """Bit for bit, of sequences and heads with and without such values, in first, middle and last blocks, over partial blocks."""

    B, H, T = 3, 2, 224
    pool, twin, table = pools(3, B, H, T, [(0, 1, 5), (1, 0, 100), (1, 1, 199)])
    args = dict(older_table=table, older_len=i32(200, 201, 33), causal=ring != "none",
                vscale=torch.tensor([0.8203125, -1.5], device=DEV) if vscale else None)
    if ring != "none":
        n = -(-(L + 20) // 32) + 1
        kl, vl = rand(8, B, L + 20, H, 128).to(DEV), rand(9, B, L + 20, H, 128).to(DEV)
        if ring == "paged":
            rtab = table_of(B, n, 4)
            local = ops.PagedKV.zeros(rtab.numel(), H, DEV)
            ops.append_paged(kl, vl, local, rtab, token0=0)
            args.update(local=local, local_table=rtab, local_ring_blocks=n, local_len=L + 20, local_start=0)
        else:
            local = ops.TiledKV.zeros(B, H, 32 * n, DEV)
            ops.pack_kv(kl.transpose(1, 2).contiguous(), vl.transpose(1, 2).contiguous(), local)
            args.update(local=local, local_len=L + 20)
    q = rand(7, B, L, G * H, 128, gain=False).to(DEV)
    got, want = (ops.prefill_attention(q, older=p, **args, **kw) for p in (pool, twin))
    assert torch.equal(got, want) and bool(got.isfinite().all())
    assert float(got.abs().max()) > 1e3  # (the large values are seen)


@pytest.mark.parametrize("host", [False, True])
@pytest.mark.parametrize("counts", [[40, 1, 200], [1, 90, 17], [70, 70, 70]])
def test_wide_tiles_of_ragged_calls(counts, host):
    pool, twin, table = pools(5, 3, 2, 416, [(0, 0, 31), (1, 1, 250), (2, 1, 400), (2, 0, 3)])
    cu = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
    q = rand(7, int(cu[-1]), 8, 128, gain=False).to(DEV)
    args = dict(older_table=table, older_len=i32(40, 300, 401), causal=False, cu_seqlens_q=torch.from_numpy(cu).to(DEV),
                max_seqlen_q=max(counts), cu_seqlens_q_host=cu if host else None, num_splits=1)
    got, want = (ops.prefill_attention(q, older=p, **args) for p in (pool, twin))
    for b, n in enumerate(counts):
        rows = slice(int(cu[b]), int(cu[b + 1]))
        if n > 16:
            assert torch.equal(got[rows], want[rows]), b
        else:  # (rows on the decode kernel: its order of sums over 8-bit pages is its own)
            a, w = got[rows].float(), want[rows].float()
            assert float((a - w).abs().max()) <= 2.0 ** -7 * float(w.abs().max())


@pytest.mark.parametrize("which", ["k", "v"])
def test_a_nan_block_beside_large_values(which):
    pool, _, table = pools(6, 1, 2, 160, [(0, 0, 70), (0, 1, 70)])
    getattr(pool, which + "_scales")[1, int(table[0, 1])] = 255
    q = rand(7, 1, 40, 8, 128, gain=False).to(DEV)
    lse = torch.zeros(1, 40, 8, device=DEV)
    got = ops.prefill_attention(q, older=pool, older_table=table, older_len=150, causal=False, lse=lse)
    assert bool(got[:, :, 4:].isnan().all()) and bool(lse[:, :, 4:].isnan().all())
    assert bool(got[:, :, :4].isfinite().all()) and bool(lse[:, :, :4].isfinite().all())


def test_what_lies_past_a_length_is_not_a_large_value():
    """Codes of tokens past the length, in a block whose power of two is large, count for nothing."""

    pool, _, table = pools(8, 1, 2, 64, [(0, 0, 40), (0, 1, 40)])
    q = rand(7, 1, 40, 8, 128, gain=False).to(DEV)
    args = dict(older=pool, older_table=table, older_len=42, causal=False)
    want = ops.prefill_attention(q, **args)
    at = np.arange(4096)
    past = torch.from_numpy((at // 16 % 64 // 16) * 8 + at % 8 >= 42 - 32).to(DEV)
    for code in (0x7f, 0x7e, 0xfe):
        b = pool.v.view(torch.uint8)
        b[:, int(table[0, 1])] = torch.where(past, torch.tensor(code, dtype=torch.uint8, device=DEV), b[:, int(table[0, 1])])
        assert torch.equal(ops.prefill_attention(q, **args), want)
