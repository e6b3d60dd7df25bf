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
