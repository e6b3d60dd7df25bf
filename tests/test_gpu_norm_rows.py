"""RMSNorm of more rows than one grid has."""

from __future__ import annotations

import pytest
import torch

from lastkv_amd import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16 = torch.bfloat16


@pytest.mark.parametrize("add", [False, True])
def test_rmsnorm_of_more_rows_than_a_grid_has(add):
    """2^24 + 3 rows: a workgroup of 256 threads each would be 2^32 threads and more.  Rows equal those of small calls."""

    rows = (1 << 24) + 3
    g = torch.Generator(device=DEV).manual_seed(1)
    x = torch.randn((1 << 12, 32), generator=g, device=DEV).to(BF16).repeat((rows >> 12) + 1, 1)[:rows]
    w = torch.randn(32, generator=g, device=DEV).to(BF16)
    residual = x.flip(0) if add else None
    at = torch.tensor([0, 1, (1 << 23) - 1, 1 << 23, (1 << 23) + 1, (1 << 24) - 1, 1 << 24, rows - 1], device=DEV)
    few = residual[at] if add else None
    want = ops.rmsnorm(x[at], w, 1e-5, residual=few)
    got = ops.rmsnorm(x, w, 1e-5, residual=residual)
    assert torch.equal(got[at], want) and got.isfinite().all()
    assert not add or torch.equal(residual[at], few)
