"""Outputs that share memory with an input, or with each other: refused on both launch paths, before any launch."""

from __future__ import annotations

import pytest
import torch

from lastkv_amd import ops

from test_gpu_mx import _gen, norm_reference, outliers, random_mx4, random_mx8, same_mx8

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16 = torch.bfloat16


@pytest.fixture(params=["native", "python"])
def path(request, monkeypatch):
    if request.param == "python":
        monkeypatch.setattr(ops, "_host", None)
        monkeypatch.setattr(ops, "_host_bound", False)
        monkeypatch.setattr(ops, "_bind_host", lambda: False)


def test_linear_outputs_over_scales_bias_or_weight(path):
    g = _gen(1)
    rows, n, k = 4, 64, 512
    pool = torch.zeros(1 << 20, dtype=torch.uint8, device=DEV)
    x = random_mx8(g, rows, k)
    w = ops.mx4_pack(*random_mx4(g, n, k))
    bias = torch.randn(n, generator=g, device=DEV).to(BF16)
    out = pool[:rows * n * 2].view(BF16).view(rows, n)
    scales = pool[448:448 + rows * k // 32].view(rows, k // 32)
    scales.copy_(x.scales)
    over_bias = pool[500:500 + 2 * n].view(BF16)
    over_bias.copy_(bias)
    size = w.data.numel()
    over_weight = pool[256:256 + size]
    over_weight.copy_(w.data)
    for call, text in ((lambda: ops.mx4_linear(ops.MX8Rows(x.data, scales), w, out=out), "scales"),
                       (lambda: ops.mx4_linear(x, w, bias=over_bias, out=out), "bias"),
                       (lambda: ops.mx4_linear(x, ops.MX4Weight(over_weight, n, k), out=out), "weight")):
        before = pool.clone()
        with pytest.raises(ValueError, match="overlap.*" + text):
            call()
        torch.cuda.synchronize()
        assert torch.equal(pool, before)
    behind = pool[512:512 + rows * k // 32].view(rows, k // 32)  # right behind the output
    behind.copy_(x.scales)
    assert torch.equal(ops.mx4_linear(ops.MX8Rows(x.data, behind), w, out=out), ops.mx4_linear(x, w))


def test_8_bit_outputs_over_their_own_scales(path):
    g = _gen(2)
    x, w = outliers(g, 4, 64), torch.ones(64, device=DEV, dtype=BF16)
    pool = torch.zeros(1024, dtype=torch.uint8, device=DEV)
    out = ops.MX8Rows(pool[:256].view(torch.float8_e4m3fn).view(4, 64), pool[250:258].view(4, 2))
    for call in (lambda: ops.rmsnorm_mx8(x, w, 1e-5, out=out), lambda: ops.silu_mul_mx8(x, x, out=out)):
        with pytest.raises(ValueError, match="data and scales"):
            call()
    assert not pool.any()
    rows = pool.view(4, 256)  # a row's data and then its scales
    out = ops.MX8Rows(rows[:, :64].view(torch.float8_e4m3fn), rows[:, 64:66])
    same_mx8(ops.rmsnorm_mx8(x, w, 1e-5, out=out), norm_reference(x, w, 1e-5))
    assert not rows[:, 66:].any()


def test_residual_over_the_weight(path):
    g = _gen(3)
    x, r = outliers(g, 4, 64), outliers(g, 5, 64)
    before = r.clone()
    with pytest.raises(ValueError, match="residual must not overlap weight"):
        ops.rmsnorm_mx8(x, r[3], 1e-5, residual=r[:4])
    assert torch.equal(r, before)
    same_mx8(ops.rmsnorm_mx8(x, r[4], 1e-5, residual=r[:4]), norm_reference(x, before[4], 1e-5, before[:4]))


def test_columns_of_one_tensor_side_by_side(path):
    """x, the residual and the output in rows of one tensor: none reaches into another's columns."""

    g = _gen(4)
    rows, k = 5, 96
    pool = torch.zeros((rows, 640), dtype=torch.uint8, device=DEV)
    x, r = pool[:, :192].view(BF16), pool[:, 192:384].view(BF16)
    x.copy_(outliers(g, rows, k))
    r.copy_(outliers(g, rows, k))
    out = ops.MX8Rows(pool[:, 384:480].view(torch.float8_e4m3fn), pool[:, 480:483])
    w = (1 + 0.3 * torch.randn(k, generator=g, device=DEV)).to(BF16)
    keep, want_r = x.clone(), (r.float() + x.float()).to(BF16)
    want = norm_reference(x, w, 1e-5, r.clone())
    same_mx8(ops.rmsnorm_mx8(x, w, 1e-5, residual=r, out=out), want)
    assert torch.equal(r, want_r) and torch.equal(x, keep) and not pool[:, 483:].any()
    want = x.double() / (1 + torch.exp(-x.double())) * r.double()
    same_mx8(ops.silu_mul_mx8(x, r, out=out), want)
    half = pool[:, 96:288].view(BF16)  # the second half of x and the first of r
    for call in (lambda: ops.rmsnorm_mx8(x, w, 1e-5, residual=half),
                 lambda: ops.silu_mul_mx8(x, r, out=ops.MX8Rows(pool[:, 352:448].view(torch.float8_e4m3fn), pool[:, 480:483]))):
        with pytest.raises(ValueError, match="overlap"):
            call()
