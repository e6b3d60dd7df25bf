"""Forks that fail half way (gpu)."""

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
