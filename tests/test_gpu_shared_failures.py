"""Forks that fail half way and beam searches over few candidates (gpu)."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from lastkv_amd import serving
from lastkv_amd.serving import LastKVServingModel

from test_gpu_llm import _tiny
from test_gpu_shared_pages import _ids, _prefill

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("shared_cache", ["bf16", "kv8"])
@pytest.mark.parametrize("failing", [1, 2])
def test_a_fork_whose_copies_fail_takes_nothing(shared_cache, failing, monkeypatch):
    _, model = _tiny(chunk=24)
    r = LastKVServingModel(model, max_batch=3, max_tokens_per_slot=256, num_splits=2, shared_cache=shared_cache)
    s, _ = _prefill(r, _ids(1, 101))
    P, calls = r.pool.pages, []
    before = (list(P._free_pages), list(P._free_slots), P.refs.copy(), P.table.copy(), P.used.copy(), r.fast._open.copy())
    copy = serving.ops.copy_pages

    def copies(*args):
        calls.append(args)
        if len(calls) == failing:
            raise RuntimeError("no copy")
        return copy(*args)

    monkeypatch.setattr(serving.ops, "copy_pages", copies)
    with pytest.raises(RuntimeError, match="no copy"):
        r.fork_sequence(s)
    assert sorted(before[0]) == sorted(P._free_pages) and sorted(before[1]) == sorted(P._free_slots)
    assert all(np.array_equal(a, b) for a, b in zip(before[2:], (P.refs, P.table, P.used, r.fast._open)))
    monkeypatch.setattr(serving.ops, "copy_pages", copy)
    twins = [r.fork_sequence(s), r.fork_sequence(s)]
    for t in range(30):
        got = r.step([(x, _ids(t, 1)) for x in (s, *twins)])
        assert torch.equal(got[0], got[1]) and torch.equal(got[0], got[2])
    for x in (s, *twins):
        r.free_sequence(x)
    assert r.pool.free_pages == r.pool.source_pages


def _masked(r, allowed, value):
    """The runner's steps with every other token's logit at `value`."""

    step = LastKVServingModel.step

    def masked(rows, *args):
        logits = step(r, rows, *args).clone()
        keep = torch.zeros(logits.shape[-1], dtype=torch.bool, device=logits.device)
        keep[allowed] = True
        return logits.masked_fill(~keep, value)

    return masked


@pytest.mark.parametrize("K,eos,allowed,steps", [(3, 11, [11, 5, 17, 40], 9), (3, 11, [5, 17, 40], 4), (2, 11, [11, 5, 17], 1),
                                                 (4, 11, [3, 4, 5, 6, 11], 6), (1, 11, [11, 7], 5)])
def test_beam_search_over_few_tokens(K, eos, allowed, steps, monkeypatch):
    """K successors are enough, where 2K candidates are looked for: the hypotheses are those of a search that gives all other tokens a
    far lower, finite logit."""

    _, model = _tiny(chunk=8, seed=23)
    out = []
    for value in (-torch.inf, -1e4):
        r = LastKVServingModel(model, max_batch=K, max_tokens_per_slot=128, num_splits=2)
        monkeypatch.setattr(r, "step", _masked(r, allowed, value))
        out.append(r.beam_search([_ids(3, 21)], num_beams=K, max_new_tokens=steps, eos_token_id=eos)[0])
        assert r.pool.free_pages == r.pool.source_pages and not r.fast._open.any()
    assert [(ids.tolist(), s) for ids, s in out[0]] == [(ids.tolist(), s) for ids, s in out[1]]
    assert len(out[0]) == K and {t for ids, _ in out[0] for t in ids[21:].tolist()} <= set(allowed)


@pytest.mark.parametrize("K,eos,allowed,steps", [(3, 11, [5, 17], 4), (3, None, [5, 17], 4), (3, 11, [11, 5, 17], 4), (3, 11, [5, 17], 1)])
def test_beam_search_over_fewer_tokens_than_beams(K, eos, allowed, steps, monkeypatch):
    _, model = _tiny(chunk=8, seed=23)
    r = LastKVServingModel(model, max_batch=K, max_tokens_per_slot=128, num_splits=2)
    monkeypatch.setattr(r, "step", _masked(r, allowed, -torch.inf))
    with pytest.raises(RuntimeError, match="fewer candidates than beams"):
        r.beam_search([_ids(3, 21)], num_beams=K, max_new_tokens=steps, eos_token_id=eos)
    assert r.pool.free_pages == r.pool.source_pages and not r.fast._open.any()
