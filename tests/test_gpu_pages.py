"""Copies of pages inside a pool (gpu; the refusals of lists need none)."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from lastkv_amd import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"


def pool_of(kind, pages, heads, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    if kind == "bf16":
        return ops.PagedKV(*(torch.randn((heads, pages, 4096), generator=g, device=DEV).bfloat16() for _ in range(2)))
    codes = [torch.randint(256, (heads, pages, 4096), generator=g, device=DEV, dtype=torch.uint8).view(torch.float8_e4m3fn)
             for _ in range(2)]
    scales = [torch.randint(256, (heads, pages), generator=g, device=DEV, dtype=torch.uint8) for _ in range(2)]
    return ops.PagedKV8(*codes, *scales)


def bytes_of(pool):
    names = ("k", "v") if isinstance(pool, ops.PagedKV) else ("k", "v", "k_scales", "v_scales")
    return [getattr(pool, n).view(torch.uint8 if n != "k" and n != "v" or isinstance(pool, ops.PagedKV8) else torch.int16) for n in names]


PAIRS = {
    "none": ([], []),
    "one": ([3], [5]),
    "to_the_last": ([0], [1099]),
    "fan_out": ([7, 7, 7], [1, 2, 3]),
    "runs": (list(range(10, 30)) + list(range(100, 137)), list(range(500, 520)) + list(range(40, 77))),
    "backwards": (list(range(50)), list(range(99, 49, -1))),
    "many_single": (list(range(0, 1000, 2)), list(range(1, 1001, 2))),  # 500 runs: two launches
}


@pytest.mark.parametrize("kind", ["bf16", "8 bits"])
@pytest.mark.parametrize("name", list(PAIRS))
@pytest.mark.parametrize("heads", [1, 3])
def test_copy_pages(name, kind, heads):
    src, dst = PAIRS[name]
    pool = pool_of(kind, 1100, heads)
    want = [t.clone() for t in bytes_of(pool)]
    for t in want:
        for a, b in zip(src, dst):
            t[:, b] = t[:, a]
    ops.copy_pages(pool, src, dst)
    assert all(torch.equal(a, b) for a, b in zip(bytes_of(pool), want))
    ops.copy_pages(pool, np.array(src, dtype=np.int64), torch.tensor(dst, dtype=torch.int32))  # again, from other lists: nothing changes
    assert all(torch.equal(a, b) for a, b in zip(bytes_of(pool), want))


def test_offsets_past_32_bits():
    pool = ops.PagedKV.zeros(150_000, 4, DEV)  # 4.9 GB a tensor
    pool.k[3, 149_998] = 1.5
    pool.v[3, 0] = 2.5
    ops.copy_pages(pool, [149_998, 0], [149_999, 149_997])
    assert bool((pool.k[3, 149_999] == 1.5).all()) and bool((pool.v[3, 149_997] == 2.5).all())
    assert not bool(pool.k[2, 149_999].any())
    del pool
    torch.cuda.empty_cache()


def test_captured_copies_replay():
    pool = pool_of("bf16", 64, 2)
    ops.copy_pages(pool, [0, 1], [10, 11])
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ops.copy_pages(pool, [0, 1], [10, 11])
    for i in range(4):
        pool.k[:, :2] = i + 1
        pool.v[:, :2] = -i - 1
        g.replay()
        torch.cuda.synchronize()
        assert bool((pool.k[:, 10:12] == i + 1).all()) and bool((pool.v[:, 10:12] == -i - 1).all())


@pytest.mark.parametrize("src,dst", [([1], [1]), ([1, 2], [5, 5]), ([1, 5], [5, 6]), ([-1], [2]), ([1], [64]), ([64], [1]), ([1, 2], [3]),
                                     ([1.5], [2]), ([[1]], [[2]]), ([1 << 40], [2])])
def test_refused_lists_change_nothing(src, dst):
    pool = pool_of("bf16", 64, 2)
    before = pool.k.clone()
    with pytest.raises((ValueError, ops._lib.LastKVNativeError)):
        ops.copy_pages(pool, src, dst)
    assert torch.equal(pool.k, before)


def test_device_lists_and_other_pools_are_refused():
    pool = pool_of("bf16", 64, 2)
    with pytest.raises(ValueError):
        ops.copy_pages(pool, torch.tensor([1], device=DEV), [2])
    with pytest.raises(ValueError):
        ops.copy_pages(ops.TiledKV.zeros(1, 1, 32, DEV), [0], [0])
