"""Long 8-bit histories: a sequence's bits go by its own keys wherever it stands in the batch, and every block is read once (gpu)."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from lastkv_amd import ops
from test_gpu_kv8 import DEV, attention64, check, history, rand, segments

pytestmark = pytest.mark.gpu


def i32(*x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


@pytest.mark.parametrize("splits", [1, 4, 8, 13])
@pytest.mark.parametrize("T", [100, 255 * 32, 256 * 32, 9999, 1024 * 32, 40000])
def test_equal_sequences_of_a_batch_have_equal_bits(T, splits):
    """One history and query at every place of a batch, and alone, beside a sequence of another length."""

    pool, table, _, _ = history(3, 1, 4, T)
    q = rand(4, 1, 16, 128, gain=False).to(DEV)
    vs = torch.tensor([0.5, 1.25, -2.0, 0.75], device=DEV)
    alone = ops.decode_attention(q, older=pool, older_table=table, older_len=T, vscale=vs, num_splits=splits)
    lens = i32(T, T, T // 3, T, T)
    got = ops.decode_attention(q.expand(5, -1, -1).contiguous(), older=pool, older_table=table.expand(5, -1).contiguous(),
                               older_len=lens, vscale=vs, num_splits=splits)
    for b in (0, 1, 3, 4):
        assert torch.equal(got[b], alone[0]), b


@pytest.mark.parametrize("L", [1, 3, 16])
@pytest.mark.parametrize("T", [9999, 40000])
def test_equal_sequences_of_a_ragged_batch_have_equal_bits(T, L):
    """Rows of a few tokens, which the decode kernel takes in a ragged call."""

    pool, table, _, _ = history(5, 1, 2, T)
    q = rand(6, L, 8, 128, gain=False).to(DEV)
    cu = np.arange(0, 4 * L + 1, L, dtype=np.int32)
    got = ops.prefill_attention(q.repeat(4, 1, 1), causal=False, older=pool, older_table=table.expand(4, -1).contiguous(), older_len=T,
                                cu_seqlens_q=torch.from_numpy(cu).to(DEV), max_seqlen_q=L, num_splits=4)
    for b in range(1, 4):
        assert torch.equal(got[b * L:(b + 1) * L], got[:L]), b


def test_a_fork_continues_as_its_parent_over_a_long_history():
    """A prompt of more than 256 blocks of history: parent and fork give the same logits for the same tokens."""

    from lastkv_amd.serving import LastKVServingModel
    from test_gpu_llm import _tiny

    _, model = _tiny(chunk=512)
    r = LastKVServingModel(model, max_batch=3, max_tokens_per_slot=9500, num_splits=4, shared_cache="kv8")
    ids = torch.randint(3, 97, (9230,), generator=torch.Generator().manual_seed(1))
    parent = r.add_sequence()
    for at in range(0, ids.numel(), 512):
        r.step([(parent, ids[at:at + 512])])
    slots = [parent, r.fork_sequence(parent)]
    slots.append(r.fork_sequence(slots[1]))
    for t in range(3):
        got = r.step([(s, ids[t:t + 1]) for s in slots])
        assert torch.equal(got[0], got[1]) and torch.equal(got[0], got[2])


@pytest.mark.parametrize("splits", [None, 1, 4, 7, 64])
@pytest.mark.parametrize("older", [[8192, 8191], [12345, 33], [32768, 32 * 1024 - 31], [34000, 32 * 1023]])
def test_long_decode_rows_to_the_weights_precision(older, splits):
    """A weight is carried as two bf16 (2^-17), and its exponential and the sums' roundings come on top: 2^-15 in all, of which a
    block left out or read twice among 1063 equal ones is thirty times as much."""

    seg, keys = segments(30, 8, 2, older, [9, 64], True)
    q = rand(31, 2, 8, 128).to(DEV)
    got = ops.decode_attention(q, num_splits=splits, **seg)
    for b in range(2):
        want, mean, err, _ = attention64(q[b:b + 1].cpu(), *keys[b], 0)
        check(got[b:b + 1], want, mean, err, 2.0 ** -15, b)


@pytest.mark.parametrize("T,splits", [(1024 * 32, 4), (1040 * 32 - 7, 5), (1500 * 32 + 1, 8), (300 * 32, 4), (1024 * 32, 1)])
def test_every_block_of_a_long_history_is_read_once(T, splits):
    """Equal keys, so that every token weighs 1 / T: the output is the mean of V, where V counts its block's number in binary
    (dim i: 1 in the blocks whose number has bit i) and dim 16 + i is 1 in every 112th block, 14 of 1500.  A block read twice or
    not at all moves one of those by a fifteenth of itself or more; every weight and sum is exact, and a bf16 output off by 2^-8."""

    nb = -(-T // 32)
    block = torch.arange(nb * 32) // 32
    v = torch.zeros(1, nb * 32, 1, 128)
    for i in range(16):
        v[0, :, 0, i] = (block >> i) & 1
    for i in range(112):
        v[0, :, 0, 16 + i] = (block % 112 == i).float()
    k = torch.ones(1, nb * 32, 1, 128)
    pool = ops.PagedKV8.zeros(nb, 1, DEV)
    table = torch.from_numpy(np.random.default_rng(1).permutation(nb).astype(np.int32))[None].to(DEV)
    src = ops.PagedKV.zeros(nb, 1, DEV)
    ops.append_paged(k.bfloat16().to(DEV), v.bfloat16().to(DEV), src, table, token0=0)
    ops.kv8_quantize(src, pool, src_table=table, dst_table=table, tokens=T)
    q = torch.ones(3, 4, 128, device=DEV).bfloat16()
    out = ops.decode_attention(q, older=pool, older_table=table.expand(3, -1).contiguous(), older_len=T, num_splits=splits)
    want = v[0, :T, 0].double().mean(0)
    off = (out.double().cpu() - want).abs()
    assert bool((off <= want * (2.0 ** -8 + 2.0 ** -15)).all()), float((off / want.clamp(min=1e-9)).max())


@pytest.mark.parametrize("host", [False, True])
@pytest.mark.parametrize("counts", [[16, 5, 1, 0], [1, 1, 8, 2], [130, 5, 1, 16]])
@pytest.mark.parametrize("T", [4000, 9001])
def test_long_ragged_rows_to_the_weights_precision(T, counts, host):
    """Rows on the decode kernel (16 tokens of a group of 4 and less) to 2^-15 of a weight, on the tiles to fp16's 2^-11 and the sum's."""

    seg, keys = segments(26, 8, 2, [T, 33, T - 1, 64], [n + 7 for n in counts], True, ring_blocks=5)
    q = rand(27, sum(counts), 8, 128).to(DEV)
    cu = np.concatenate(([0], np.cumsum(counts))).astype(np.int32)
    got = ops.prefill_attention(q, cu_seqlens_q=torch.from_numpy(cu).to(DEV), max_seqlen_q=max(counts),
                                cu_seqlens_q_host=cu if host else None, **seg)
    for b, n in enumerate(counts):
        if n:
            rows = slice(int(cu[b]), int(cu[b + 1]))
            want, mean, err, _ = attention64(q[rows].cpu(), *keys[b], n)
            check(got[rows], want, mean, err, 2.0 ** -15 if n <= 16 else 2.0 ** -10, (T, b))


@pytest.mark.parametrize("T", [0, 1, 31, 32])
@pytest.mark.parametrize("L", [1, 2, 4])
def test_shortest_histories_to_the_weights_precision(T, L):
    seg, keys = segments(36, 16, 1, [T, 0], [L, L], True)
    q = rand(37, 2, L, 16, 128).to(DEV)
    got = ops.prefill_attention(q, **seg) if L > 1 else ops.decode_attention(q[:, 0].contiguous(), **seg)[:, None]
    for b in range(2):
        want, mean, err, _ = attention64(q[b].cpu(), *keys[b], L)
        check(got[b], want, mean, err, 2.0 ** -15, (T, L, b))
