"""What a shared history in 8 bits takes, and the copies of K that prefill calls over it make (gpu)."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from lastkv_amd import ops
from lastkv_amd.serving import LastKVServingModel

from test_gpu_kv8 import DEV, attention64, check, history, rand
from test_gpu_llm import _tiny
from test_gpu_shared_pages import _ids, _prefill

pytestmark = pytest.mark.gpu


def i32(*x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def _bytes(r):
    P, tensors = r.pool, [r.pool.pool.k, r.pool.pool.v, r.fast._prefill_ws]
    if P.kv8:
        tensors += [P.shared.k, P.shared.v, P.shared.k_scales, P.shared.v_scales]
    return sum(t.numel() * t.element_size() for t in tensors)


def test_short_steps_and_one_long_row_reserve_what_they_need():
    """Steps of short rows reserve what they do over bf16 pages, a prompt's piece beside them one row's copies more."""

    _, model = _tiny(chunk=128)
    for long in (1, 3):
        ws = []
        for kind in ("bf16", "kv8"):
            r = LastKVServingModel(model, max_batch=4, max_tokens_per_slot=1024, num_splits=2, shared_cache=kind)
            group = r.fast.num_q_heads // r.pool.kv_heads
            few, many = 64 // group, 64 // group + 1
            slots = [_prefill(r, _ids(i, 640))[0] for i in range(4)]
            r.fast._prefill_ws = r.fast._prefill_ws[:0]
            sizes = []
            r.step([(slots[0], _ids(1, few)), (slots[1], _ids(2, 1)), (slots[2], _ids(2, few))])
            sizes.append(r.fast._prefill_ws.numel())
            r.step([(s, _ids(1, many if i < long else 1)) for i, s in enumerate(slots)])
            sizes.append(r.fast._prefill_ws.numel())
            ws.append(sizes)
        width = (640 - 128) // 32
        assert ws[1][0] == ws[0][0]
        assert ws[1][1] - ws[0][1] == ops.kv8_copy_bytes(long, r.pool.kv_heads, 32 * width, 4)


def test_8_bits_and_a_prompt_piece_take_less_than_bf16():
    """Sequences that fill their pages, prefilled one at a time and all at once, the pools and the workspace together: half of the
    pages goes, the staging pages come on top, and a copy of K of the rows in one step (as much as the codes; all at once, the
    staging pages are all that is left of the difference)."""

    _, model = _tiny(chunk=128)
    for rows in (1, 4):
        total = []
        for kind in ("bf16", "kv8"):
            r = LastKVServingModel(model, max_batch=4, max_tokens_per_slot=4096, num_splits=2, shared_cache=kind)
            slots = [r.add_sequence() for _ in range(4)]
            for first in range(0, 4, rows):
                for at in range(0, 4096, 128):
                    r.step([(s, _ids(at, 128)) for s in slots[first:first + rows]])
            total.append(_bytes(r))
        P = r.pool
        saved = P.kv_heads * P.source_pages * (8192 - 2)  # (and two scale bytes a page)
        spent = P.kv_heads * (4 * P.stage_blocks * 16384 + 8196) + ops.kv8_copy_bytes(rows, P.kv_heads, 4096, 4)  # (and a scratch page)
        assert total[0] - total[1] >= saved - spent and (rows == 4 or saved - spent > total[0] // 5), rows


@pytest.mark.parametrize("host", [False, True])
@pytest.mark.parametrize("counts", [[1, 1, 40, 2, 17, 1, 300], [17, 1, 18], [200, 0, 1, 90], [1] * 70 + [33] + [1] * 70 + [20, 40]])
def test_ragged_copies_go_to_their_sequences(counts, host):
    """Long rows anywhere among short ones, over histories of different lengths, in a workspace of just the size that is asked for."""

    B = len(counts)
    rng = np.random.default_rng(B)
    older = [int(n) for n in rng.integers(0, 200, B)]
    pool, table, k, v = history(B, B, 2, 224)
    cu = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
    q = rand(3, int(cu[-1]), 8, 128, gain=False)
    tiles = sum(n > 16 for n in counts) if host else min(B, sum(counts) // 17)
    need = (ops.prefill_workspace_bytes(B, 2, 224, 0) + ops.ragged_split_state_bytes(B, 8, 2, max(counts), 1, 256)
            + ops.kv8_copy_bytes(tiles, 2, 224, B))
    ws = torch.full((need + 4096,), 0xa5, dtype=torch.uint8, device=DEV)
    out = ops.prefill_attention(q.to(DEV), older=pool, older_table=table, older_len=i32(*older), causal=False, num_splits=1,
                                cu_seqlens_q=torch.from_numpy(cu).to(DEV), max_seqlen_q=max(counts),
                                cu_seqlens_q_host=cu if host else None, workspace=ws[:need])
    assert bool((ws[need:] == 0xa5).all())
    for b, n in enumerate(counts):
        if n and (n > 1 or b % 9 == 0):
            want, mean, err, _ = attention64(q[cu[b]:cu[b + 1]], k[b, :, :older[b]].cpu(), v[b, :, :older[b]].cpu(), 0)
            check(out[cu[b]:cu[b + 1]], want, mean, err, 2.0 ** -10, b)


def test_offsets_that_change_between_replays():
    """A captured ragged call without host offsets: other sequences are the long ones in every replay."""

    B, T = 4, 120
    pool, table, _, _ = history(11, B, 2, 256)
    q = rand(3, T, 8, 128, gain=False).to(DEV)
    cu = i32(0, 1, 41, 42, T)
    out, ws = torch.empty_like(q), torch.empty(1 << 24, dtype=torch.uint8, device=DEV)
    lens = i32(256, 100, 3, 77)
    call = lambda **kw: ops.prefill_attention(q, older=pool, older_table=table, older_len=lens, causal=False, cu_seqlens_q=cu,
                                              max_seqlen_q=100, **kw)
    call(out=out, workspace=ws)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        call(out=out, workspace=ws)
    for offsets in ([0, 1, 41, 42, T], [0, 90, 91, 92, T], [0, 30, 60, 90, T], [0, 5, 5, 104, T], [0, 1, 2, 20, T]):
        cu.copy_(i32(*offsets))
        ws.fill_(0xff)
        out.zero_()
        g.replay()
        torch.cuda.synchronize()
        got = out.clone()
        assert torch.equal(got, call()), offsets


def test_offsets_that_the_call_has_no_room_for_stay_inside_it():
    """Device offsets that name more long sequences than the rows allow (they overlap): nothing is written behind the workspace."""

    B, T = 6, 40
    pool, table, _, _ = history(12, B, 2, 256)
    q = rand(3, T, 8, 128, gain=False).to(DEV)
    args = dict(older=pool, older_table=table, older_len=256, causal=False, max_seqlen_q=T, num_splits=1)
    need = (ops.prefill_workspace_bytes(B, 2, 256, 0) + ops.ragged_split_state_bytes(B, 8, 2, T, 1, 256)
            + ops.kv8_copy_bytes(T // 17, 2, 256, B))
    ws = torch.full((need + (1 << 22),), 0xa5, dtype=torch.uint8, device=DEV)
    ops.prefill_attention(q, cu_seqlens_q=i32(0, T, 0, T, 0, T, 0), workspace=ws[:need], **args)
    torch.cuda.synchronize()
    assert bool((ws[need:] == 0xa5).all())


@pytest.mark.parametrize("length", ["device", "fixed"])
@pytest.mark.parametrize("ring", ["tiled", "paged"])
@pytest.mark.parametrize("counts,kw", [([40, 1, 17, 90], dict()), ([3, 16, 0, 9], dict(tile_waves=4)), ([1, 5], dict(tile_waves=8)),
                                       ([3, 70, 16], dict(tile_waves=8))])
def test_ragged_tiles_beside_rings_of_either_kind(counts, kw, ring, length):
    """Rows on the tiles, short ones too where `tile_waves` puts a call of those alone there, equal the call over bf16 pages of the same
    values in every bit; rings in slots of any order."""

    B, H, T, W = len(counts), 2, 200, 4
    pool, table, k, v = history(21, B, H, 224)
    twin = ops.PagedKV.zeros(table.numel(), H, DEV)
    ops.append_paged(k.transpose(1, 2).contiguous(), v.transpose(1, 2).contiguous(), twin, table, token0=0)
    kl, vl = rand(22, B, 32 * W, H, 128).to(DEV), rand(23, B, 32 * W, H, 128).to(DEV)
    order = np.random.default_rng(B).permutation(B).astype(np.int32)
    local = [n + 5 for n in counts]
    args = dict(local_len=i32(*local), local_start=i32(*[7 * b for b in range(B)]), causal=True, num_splits=1,
                older_table=table, older_len=T if length == "fixed" else i32(*[T - 63 * b for b in range(B)]),
                vscale=torch.tensor([0.8203125, -1.5], device=DEV))
    if ring == "tiled":
        cache = ops.TiledKV.zeros(B, H, 32 * W, DEV)
        ops.pack_kv(kl.transpose(1, 2).contiguous(), vl.transpose(1, 2).contiguous(), cache)
        args.update(local=cache, local_slot=torch.from_numpy(order).to(DEV))
    else:
        rtab = torch.from_numpy((order[:, None] * W + np.arange(W)).astype(np.int32)).to(DEV)
        local_pool = ops.PagedKV.zeros(B * W, H, DEV)
        ops.append_paged(kl, vl, local_pool, rtab, token0=0)
        args.update(local=local_pool, local_table=rtab, local_ring_blocks=W)
    cu = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
    q = rand(24, int(cu[-1]), 8, 128, gain=False).to(DEV)
    for host in (None, cu):
        got, want = (ops.prefill_attention(q, older=p, cu_seqlens_q=torch.from_numpy(cu).to(DEV), max_seqlen_q=max(counts),
                                           cu_seqlens_q_host=host, **args, **kw) for p in (pool, twin))
        for b, n in enumerate(counts):
            if n > 16 or max(counts) <= 16:
                assert torch.equal(got[cu[b]:cu[b + 1]], want[cu[b]:cu[b + 1]]), b
