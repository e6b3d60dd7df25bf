"""mx4_linear(exact=True): 8-bit rows with exact products and fp32 sums at any number of rows."""

from __future__ import annotations

import pytest
import torch

from lastkv_amd import ops

from test_gpu_mx import _gen, mx4_values, mx8_values, random_mx4, random_mx8

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("m", [1, 16, 17, 300])
def test_products_that_cancel(m):
    """256 - 256 + 2^-b among eight neighbouring columns of a weight of ones, in a call with enough work for tiles."""

    n = 16400
    w = ops.mx4_pack(torch.full((n, 256), 0x22, dtype=torch.uint8, device=DEV),
                     torch.full((n, 16), 127, dtype=torch.uint8, device=DEV))
    for at, b in ((2, 5), (2, 6), (7, 9), (300, 9)):
        x = torch.zeros((m, 512), device=DEV)
        x[:, 0], x[:, 1], x[:, at] = 256, -256, 2.0 ** -b
        x = ops.MX8Rows(x.to(torch.float8_e4m3fn), torch.full((m, 16), 127, dtype=torch.uint8, device=DEV))
        assert ops.mx4_linear(x, w, exact=True).eq(2.0 ** -b).all(), (at, b)


@pytest.mark.parametrize("m,n,k", [(5, 100, 96), (40, 28700, 160), (1030, 8001, 544), (1000, 6144, 1024)])
def test_sums_in_fp32(m, n, k):
    """Within K fp32 additions of the sum of magnitudes (2^-24 each) and one rounding to bf16 (2^-8 of the value covers
    half a step), without the fixed point's share; the bias and out go with it."""

    g = _gen(m + n)
    codes, scales = random_mx4(g, n, k)
    x, w = random_mx8(g, m, k), ops.mx4_pack(codes, scales)
    bias = torch.randn(n, generator=g, device=DEV).bfloat16()
    out = torch.empty((m, n), device=DEV, dtype=torch.bfloat16)
    assert ops.mx4_linear(x, w, bias, out, exact=True) is out
    xv, wv = mx8_values(x).to(DEV), mx4_values(codes, scales).to(DEV)
    want = xv @ wv.t() + bias.double()
    tol = 2.0 ** -8 * want.abs() + (k + 1) * 2.0 ** -24 * (xv.abs() @ wv.abs().t() + bias.double().abs())
    assert bool(((out.double() - want).abs() <= tol).all())
    assert torch.equal(out, ops.mx4_linear(ops.mx8_unpack(x), w, bias))
    y = ops.mx8_unpack(x)
    assert torch.equal(ops.mx4_linear(y, w, exact=True), ops.mx4_linear(y, w))
