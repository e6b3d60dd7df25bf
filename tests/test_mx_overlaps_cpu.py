"""Whether two tensors share memory, as the low-bit operators decide it, against the sets of their bytes."""

from __future__ import annotations

import itertools

import torch

from lastkv_amd import ops


def _bytes(t):
    at = [t.data_ptr()]
    for n, st in zip(t.shape, t.stride()):
        at = [a + i * st * t.element_size() for a in at for i in range(n)]
    return {a + b for a in at for b in range(t.element_size())}


def test_address_ranges_and_column_slices():
    pool = torch.zeros(4096, dtype=torch.uint8)
    wide = pool[:1024].view(torch.bfloat16).view(4, 128)
    parts = [wide[:, :64], wide[:, 64:], wide[:, 32:96], wide[:2, :64], wide[1:3, 64:], wide[:1, :64], wide[1:2, :64],
             pool[1024:1536].view(torch.bfloat16).view(4, 64), pool[1536:1600].view(torch.bfloat16),
             wide.view(torch.uint8)[:, 128:192], wide.view(torch.uint8)[:, 192:194], wide.view(2, 2, 128)[..., 64:],
             pool[:960].view(4, 240)[:, 128:192]]
    sides = 0
    for a, b in itertools.product(parts, parts):
        shared = bool(_bytes(a) & _bytes(b))
        assert not shared or ops._overlap(a, b)
        if a.shape[:-1].numel() == b.shape[:-1].numel():
            beside = ops._beside(a, b)
            assert not (shared and beside)
            sides += beside and ops._overlap(a, b)
    assert ops._beside(parts[0], parts[1]) and ops._beside(parts[1], parts[0]) and ops._beside(parts[9], parts[10])
    assert not ops._beside(parts[0], parts[2]) and not ops._beside(parts[0], parts[0])
    assert sides >= 8


def test_neighbours_do_not_overlap():
    pool = torch.zeros(256, dtype=torch.uint8)
    assert not ops._overlap(pool[:64], pool[64:]) and ops._overlap(pool[:65], pool[64:]) and not ops._overlap(pool[:0], pool)
