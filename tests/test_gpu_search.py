"""Beam search's selection against its formula in 64 bits (gpu)."""

from __future__ import annotations

import math

import pytest
import torch

from lastkv_amd import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"


def reference(logits, scores, count):
    """Scores, beams and tokens in 64 bits, ties to the lowest index; what is no candidate is (-inf, -1, -1)."""

    x = logits.double().cpu()
    B, K, V = x.shape
    total = (scores.double().cpu()[..., None] + (x - torch.logsumexp(x, -1, keepdim=True))).reshape(B, K * V)
    total = torch.where(total.isnan(), -math.inf, total)
    best, index = torch.sort(total, dim=1, descending=True, stable=True)
    if K * V < count:
        best = torch.nn.functional.pad(best, (0, count - K * V), value=-math.inf)
        index = torch.nn.functional.pad(index, (0, count - K * V))
    best, index = best[:, :count], index[:, :count]
    none = best == -math.inf
    return best, torch.where(none, -1, index // V), torch.where(none, -1, index % V)


def check(logits, scores, count, **kw):
    got = ops.beam_select(logits, scores, count, **kw)
    want = reference(logits, scores, count)
    assert torch.equal(got[1].cpu().long(), want[1]) and torch.equal(got[2].cpu().long(), want[2])
    # fp32's rounding (2^-24 of the value) and the sums of exponentials: a thread adds up to 32 in fp32, each off by a few 2^-24
    # of itself, which the sum's logarithm carries over as 40 * 2^-24 at most
    a, b = got[0].double().cpu(), want[0]
    fin = torch.isfinite(b)
    assert bool((a[~fin] == -math.inf).all())
    assert bool(((a - b).abs()[fin] <= b.abs()[fin] * 2.0 ** -24 + 40 * 2.0 ** -24).all())
    return got


def logits_of(seed, B, K, V, dtype):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (3 * torch.randn((B, K, V), generator=g, device=DEV)).to(dtype)


def scores_of(seed, B, K):
    return -10 * torch.rand((B, K), generator=torch.Generator().manual_seed(seed)).to(DEV)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("B,K,V,count", [(1, 1, 1, 1), (1, 1, 1, 5), (2, 3, 7, 6), (1, 4, 2047, 8), (3, 2, 2048, 64), (2, 5, 8193, 10),
                                         (1, 64, 500, 64), (1, 8, 50257, 16), (4, 12, 32001, 24), (33, 8, 9000, 16)])
def test_against_64_bits(B, K, V, count, dtype):
    check(logits_of(V, B, K, V, dtype), scores_of(K, B, K), count)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_ties_go_to_the_lowest_index(dtype):
    """Equal logits everywhere (more of them than one pass holds), equal beams, a few values over and over."""

    x = torch.zeros((2, 3, 9001), dtype=dtype, device=DEV)
    check(x, torch.zeros(2, 3, device=DEV), 64)
    y = (logits_of(1, 2, 1, 5000, torch.float32).round() / 2).to(dtype).expand(2, 4, 5000).contiguous()
    check(y, torch.full((2, 4), -1.25, device=DEV), 40)
    z = x.clone()
    z[:, 1, 8999] = 1
    z[:, :, 5] = 1
    check(z, torch.zeros(2, 3, device=DEV), 20)


def test_few_threads_hold_all_the_best():
    """Descending logits: the best lie in the first pieces."""

    x = -torch.arange(20000, device=DEV).float()[None, None] * 1e-3
    check(x.contiguous(), torch.zeros(1, 1, device=DEV), 64)
    check(x.to(torch.bfloat16), torch.zeros(1, 1, device=DEV), 64)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_masks_and_dead_beams(dtype):
    x = logits_of(3, 4, 4, 4000, dtype)
    s = scores_of(2, 4, 4)
    x[0, :, 10:] = -math.inf           # ten tokens allowed: 40 candidates
    x[1, 1, 77] = math.nan             # that beam drops out
    x[1, 2, 5] = math.inf              # and that one
    x[2] = -math.inf                   # none at all
    x[3, 0, 1:] = -math.inf            # one certain token
    s[3, 1:] = -math.inf               # a first step: one beam
    got = check(x, s, 50)
    assert got[1][2].eq(-1).all() and got[1][3].tolist() == [0] + [-1] * 49
    s[0, 0] = math.nan
    check(x, s, 50)
    s[0, 1] = math.inf                 # (nor is one whose score is +inf)
    got = ops.beam_select(x, s, 50)
    assert set(got[1][0].tolist()) == {2, 3, -1} and int(got[1][0].eq(-1).sum()) == 30


def test_one_beam_keeps_the_order_of_its_logits():
    """Logits that a score of 64 bits cannot tell apart: the greater one first all the same."""

    x = (torch.randperm(3000, generator=torch.Generator().manual_seed(1)) * 2.0 ** -40).to(DEV)[None, None].contiguous()
    got = ops.beam_select(x, torch.full((1, 1), -1e30, device=DEV), 20)
    assert got[2][0].tolist() == x[0, 0].argsort(descending=True)[:20].tolist()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_large_values_and_lowest_values(dtype):
    x = logits_of(4, 2, 2, 3001, dtype)
    x[0] *= 1e4
    x[1, :, ::3] = torch.finfo(dtype).min
    check(x, torch.zeros(2, 2, device=DEV), 12)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("lead", [1, 3, 4, 7])
def test_rows_at_any_alignment(dtype, lead):
    big = logits_of(5, 3, 5, 4099, dtype)
    view = big[:, 1:4, lead:lead + 4083]
    check(view, scores_of(1, 3, 3), 9)
    check(big.transpose(0, 1)[:, :, lead:], scores_of(1, 5, 3), 9)
    whole = scores_of(8, 3, 7)
    check(view, whole[:, 2:5], 9)


def test_two_calls_agree_and_a_graph_replays():
    x, s = logits_of(6, 2, 4, 33000, torch.bfloat16), scores_of(3, 2, 4)
    a, b = ops.beam_select(x, s, 8), ops.beam_select(x, s, 8)
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    ws = torch.empty(ops.beam_workspace_bytes(2, 4, 33000, 8), dtype=torch.uint8, device=DEV)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = ops.beam_select(x, s, 8, workspace=ws)
    for i in range(4):
        x.copy_(logits_of(20 + i, 2, 4, 33000, torch.bfloat16))
        ws.fill_(255)
        g.replay()
        torch.cuda.synchronize()
        want = ops.beam_select(x, s, 8)
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(out, want))


def test_refusals():
    x, s = logits_of(7, 1, 2, 100, torch.float32), scores_of(1, 1, 2)
    err = (ValueError, ops._lib.LastKVNativeError)
    for a in ((x.half(), s, 2), (x.cpu(), s, 2), (x[0], s, 2), (x.transpose(1, 2), s, 2), (x, s[:, :1], 2), (x, s.double(), 2),
              (x, s.cpu(), 2), (x, s, 0), (x, s, 65), (x, s, 2.0), (x[:, :, :0], s, 2)):
        with pytest.raises(err):
            ops.beam_select(*a)
    with pytest.raises(err):
        ops.beam_select(x, s, 2, workspace=torch.empty(8, dtype=torch.uint8, device=DEV))
    with pytest.raises(err):
        ops.beam_select(x.expand(1, 2, 100).repeat(1, 33, 1), scores_of(1, 1, 66), 2)
