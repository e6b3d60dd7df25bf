"""8-bit outputs where fp32's range ends before the operator's: still the bits of the 64-bit value."""

from __future__ import annotations

import pytest
import torch

from lastkv_amd import ops

from test_gpu_mx import _gen, norm_reference, same_mx8

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16 = torch.bfloat16


@pytest.mark.parametrize("low", [-133, -130, -126, -120])
@pytest.mark.parametrize("row", [0, 8, 30])
def test_rmsnorm_mx8_of_tiny_values_under_large_weights(low, row):
    """A row of 2^row whose other values are near 2^low: value / rms falls below fp32's normal range (2^-126), the
    weight of about 2^127 brings it back."""

    g = _gen(row - low)
    rows, k = 64, 1024
    x = torch.randn((rows, k), generator=g, device=DEV).double() * 2.0 ** low * 4
    x[:, :32] = torch.randn((rows, 32), generator=g, device=DEV).double() * 2.0 ** row * 4
    x = x.to(BF16)
    w = torch.ldexp(1 + torch.rand(k, generator=g, device=DEV), torch.tensor(126.0, device=DEV)).to(BF16)
    w[:32] = 1
    assert (x[:, 32:] != 0).any() and torch.isfinite(w).all()
    same_mx8(ops.rmsnorm_mx8(x, w, 1e-5), norm_reference(x, w, 1e-5))


@pytest.mark.parametrize("add", [False, True])
def test_rmsnorm_mx8_of_more_rows_than_a_grid_has(add):
    """2^24 + 3 rows: a workgroup of 256 threads each would be 2^32 threads and more."""

    rows = (1 << 24) + 3
    x = torch.randn((1 << 12, 32), generator=_gen(5), device=DEV).to(BF16).repeat((rows >> 12) + 1, 1)[:rows]
    w = torch.ones(32, device=DEV, dtype=BF16)
    residual = x.flip(0) if add else None
    at = torch.tensor([0, 1, (1 << 23) - 1, 1 << 23, (1 << 23) + 1, (1 << 24) - 1, 1 << 24, rows - 1], device=DEV)
    want = norm_reference(x[at], w, 1e-5, residual[at] if add else None)
    sums = (residual[at].float() + x[at].float()).to(BF16) if add else None
    q = ops.rmsnorm_mx8(x, w, 1e-5, residual=residual)
    same_mx8(ops.MX8Rows(q.data[at], q.scales[at]), want)
    assert not add or torch.equal(residual[at], sums)
