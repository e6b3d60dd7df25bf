"""The low-bit operators without a GPU: refusals of the C ABI and of ops.py before any launch, fake shapes of the
custom operators."""

from __future__ import annotations

import ctypes

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import lastkv_amd.torch_ops  # noqa: F401  (registers torch.ops.lastkv.*)
from lastkv_amd import _lib, ops


def _norm(**kw):
    a = _lib.NormMx8Args()
    a.struct_size = ctypes.sizeof(a)
    a.rows, a.hidden, a.x = 1, 64, 16
    a.weight = a.out = a.scales = 16
    for k, v in kw.items():
        setattr(a, k, v)
    return _lib.load().lkv_rmsnorm_mx8(ctypes.byref(a), None), _lib.load().lkv_last_error()


@pytest.mark.parametrize("kw,message", [
    (dict(struct_size=8), b"size mismatch"), (dict(rows=-1), b"rows"), (dict(hidden=40), b"multiple of 32"),
    (dict(hidden=0), b"multiple of 32"), (dict(hidden=16416), b"up to 16384"), (dict(x=None), b"null"),
    (dict(scales=None), b"null"), (dict(x=24), b"aligned"), (dict(residual=8), b"aligned"), (dict(out=20), b"aligned"),
    (dict(x_stride=12), b"multiples of 8"), (dict(out_stride=4), b"multiples of 8"),
    (dict(rows=2, x_stride=64, out_stride=56, scale_stride=2), b"overlap"),
    (dict(rows=2, x_stride=64, out_stride=64, scale_stride=1), b"overlap"),
    (dict(rows=2, x_stride=64, out_stride=64, scale_stride=2, residual=16), b"overlap")])
def test_norm_refusals(kw, message):
    st, text = _norm(**kw)
    assert st == 1 and message in text, text


def test_norm_without_rows_launches_nothing():
    assert _norm(rows=0)[0] == 0


def _linear(**kw):
    a = _lib.Mx4LinearArgs()
    a.struct_size = ctypes.sizeof(a)
    a.rows, a.out_features, a.in_features, a.x_stride, a.out_stride = 1, 16, 64, 64, 16
    a.x = a.weight = a.out = 16
    for k, v in kw.items():
        setattr(a, k, v)
    return _lib.load().lkv_mx4_linear(ctypes.byref(a), None), _lib.load().lkv_last_error()


@pytest.mark.parametrize("kw,message", [
    (dict(struct_size=8), b"size mismatch"), (dict(rows=-1), b"rows"), (dict(rows=(1 << 20) + 1), b"rows"),
    (dict(in_features=48), b"multiple of 32"), (dict(in_features=0), b"multiple of 32"), (dict(out_features=0), b"1 to 2^24"),
    (dict(in_features=(1 << 20) + 32), b"up to 2^20"), (dict(x_format=2), b"x_format"), (dict(kernel=3), b"kernel"), (dict(x=None), b"null"),
    (dict(weight=None), b"null"), (dict(out=None), b"null"), (dict(x_format=1), b"x_scales"), (dict(x_scales=16), b"x_scales"),
    (dict(x=24), b"aligned"), (dict(weight=8), b"aligned"), (dict(rows=2, x_stride=68), b"aligned"),
    (dict(rows=2, x_format=1, x_scales=16, x_stride=72), b"aligned"), (dict(rows=2, x_stride=1 << 24), b"2^21"), (dict(rows=2, x_stride=-8), b"2^21"),
    (dict(rows=2, x_format=1, x_scales=16, x_scale_stride=1 << 32), b"x_scale_stride"),
    (dict(rows=2, x_format=1, x_scales=16, x_scale_stride=-1), b"x_scale_stride"), (dict(rows=2, out_stride=15), b"overlap")])
def test_linear_refusals(kw, message):
    st, text = _linear(**kw)
    assert st == 1 and message in text, text


def test_linear_without_rows_launches_nothing():
    assert _linear(rows=0)[0] == 0


def test_other_refusals_and_sizes():
    lib = _lib.load()
    assert lib.lkv_silu_mul_mx8(16, 64, 16, 64, 16, 64, 16, 2, 1, 40, None) == 1 and b"multiple of 32" in lib.lkv_last_error()
    assert lib.lkv_silu_mul_mx8(16, 64, 24, 64, 16, 64, 16, 2, 1, 64, None) == 1 and b"aligned" in lib.lkv_last_error()
    assert lib.lkv_silu_mul_mx8(16, 64, 16, 64, 16, 0, 16, 2, 2, 64, None) == 1 and b"overlap" in lib.lkv_last_error()
    assert lib.lkv_mx8_unpack(16, 64, 16, 2, 16, 0, 2, 64, None) == 1 and b"overlap" in lib.lkv_last_error()
    assert lib.lkv_mx8_unpack(16, 64, None, 2, 16, 64, 1, 64, None) == 1 and b"null" in lib.lkv_last_error()
    assert lib.lkv_mx8_unpack(16, 60, 16, 2, 16, 64, 1, 64, None) == 1 and b"multiples of 8" in lib.lkv_last_error()
    for call in (lambda: lib.lkv_mx4_pack(16, 32, 16, 2, 16, 40, 16, None), lambda: lib.lkv_mx4_quantize(16, 64, 0, 64, 16, None),
                 lambda: lib.lkv_mx4_unpack(16, 16, 48, 16, 64, None)):
        assert call() == 1 and b"multiple of 32" in lib.lkv_last_error()
    assert lib.lkv_mx4_weight_bytes(16, 512) == 4352 and lib.lkv_mx4_weight_bytes(17, 544) == 2 * (2 * 4352 + 256)
    assert lib.lkv_mx4_weight_bytes(0, 512) == 0


def test_cpu_tensors_and_shapes_are_refused():
    bf = dict(dtype=torch.bfloat16)
    x, w = torch.zeros((2, 64), **bf), torch.zeros(64, **bf)
    for call in (lambda: ops.rmsnorm_mx8(x, w, 1e-5), lambda: ops.silu_mul_mx8(x, x), lambda: ops.mx4_quantize(x),
                 lambda: ops.MX8Rows.empty((2, 64), "cpu"), lambda: ops.MX4Weight(torch.zeros(4352, dtype=torch.uint8), 16, 64),
                 lambda: ops.mx4_pack(torch.zeros((4, 32), dtype=torch.uint8), torch.zeros((4, 2), dtype=torch.uint8))):
        with pytest.raises(ValueError, match="GPU"):
            call()
    with pytest.raises(ValueError, match="MX4Weight"):
        ops.mx4_linear(x, x)
    with pytest.raises(ValueError, match="MX8Rows"):
        ops.mx8_unpack(x)


def test_custom_operators_fake_shapes():
    with FakeTensorMode():
        x = torch.empty((3, 5, 64), dtype=torch.bfloat16)
        w = torch.empty(64, dtype=torch.bfloat16)
        for data, scales in (torch.ops.lastkv.rmsnorm_mx8(x, w, 1e-5), torch.ops.lastkv.silu_mul_mx8(x, x),
                             torch.ops.lastkv.add_rmsnorm_mx8(x, x, w, 1e-5)):
            assert data.shape == x.shape and data.dtype == torch.float8_e4m3fn
            assert scales.shape == (3, 5, 2) and scales.dtype == torch.uint8
        assert torch.ops.lastkv.mx8_unpack(data, scales).dtype == torch.bfloat16
        weight = torch.empty(4352, dtype=torch.uint8)
        assert torch.ops.lastkv.mx4_linear(x, weight, 10).shape == (3, 5, 10)
        y = torch.ops.lastkv.mx4_linear_mx8(data, scales, weight, 10)
        assert y.shape == (3, 5, 10) and y.dtype == torch.bfloat16
    schema = torch.ops.lastkv.add_rmsnorm_mx8.default._schema
    assert {a.name for a in schema.arguments if a.alias_info is not None and a.alias_info.is_write} == {"residual"}
