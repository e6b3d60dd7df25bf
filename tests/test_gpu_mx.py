"""The low-bit operators against 64-bit references.

8-bit outputs are correctly rounded from the operator's real value, so they equal the 64-bit reference's bit for bit
(its own error, about 1e-15 relative, is 10^-13 of a rounding step).  Products: bf16 x e2m1 and e4m3 x e2m1 terms are
exact in fp32; K of them and the wave sums are added in fp32, each addition off by at most 2^-24 of the running
magnitude, which sum |x w| bounds: K * 2^-24 * sum |x w| covers any order; the result is rounded to bf16 once (2^-8
of a value at most half a step = 2^-9 times its power of two, so 2^-8 relative covers it).
The tile kernel's MX8 rows go through the scaled matrix instruction, which first adds the products of 8 neighbouring
columns in fixed point: bits below 2^-13 of the largest 2^(ex + ew), the powers of two of a product's factors, are dropped
(test_mx8_products_that_cancel pins it), so each of the other 7 products loses less than 2^-13 times the
group's largest product, which (largest |x|) * (largest |w|) of the group bounds.
"""

from __future__ import annotations

import ctypes
import math

import pytest
import torch

from lastkv_amd import _lib, ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16 = torch.bfloat16
E2M1 = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, 0, -0.5, -1, -1.5, -2, -3, -4, -6], dtype=torch.float64)
E4M3 = torch.tensor([(m / 8 * 2.0 ** -6) if e == 0 else (1 + m / 8) * 2.0 ** (e - 7) for e in range(16) for m in range(8)][:127],
                    dtype=torch.float64)


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _pow2(e):
    """2^e in 64 bits, exact (e an integer tensor)."""

    return torch.ldexp(torch.ones_like(e, dtype=torch.float64).cpu(), e.cpu()).to(e.device)


def mx8_reference(y):
    """(values' codes, scale bytes) of 64-bit rows: the smallest power of two that holds a block, nearest, ties to even."""

    shape = y.shape
    b = y.reshape(-1, 32).cpu()
    bad = ~torch.isfinite(b).all(1)
    b = torch.where(bad[:, None], torch.zeros_like(b), b)
    amax = b.abs().amax(1)
    m, e = torch.frexp(amax)
    byte = torch.where(amax > 0, (e - 9 + (m > 0.875).to(e.dtype) + 127).clamp(min=0), torch.zeros_like(e))
    v = torch.ldexp(b, (127 - byte)[:, None])
    mids = (E4M3[1:] + E4M3[:-1]) / 2
    lo, hi = torch.bucketize(v.abs(), mids), torch.bucketize(v.abs(), mids, right=True)
    code = torch.where(lo % 2 == 0, lo, hi) | (torch.signbit(v).long() << 7)
    byte = torch.where(bad, torch.full_like(byte, 255), byte)
    code = torch.where(bad[:, None], torch.zeros_like(code), code)
    return code.to(torch.uint8).reshape(shape), byte.to(torch.uint8).reshape(*shape[:-1], shape[-1] // 32)


def mx8_values(rows):
    code = rows.data.view(torch.uint8).cpu().long()
    table = torch.cat([E4M3, torch.tensor([math.nan], dtype=torch.float64)])
    v = table[code & 127] * torch.where(code >= 128, -1.0, 1.0).double()
    e = rows.scales.cpu().int()
    s = torch.where(e == 255, torch.tensor(math.nan, dtype=torch.float64), _pow2(e - 127))
    return v * s.repeat_interleave(32, -1)


def mx4_values(codes, scales):
    c = torch.stack((codes & 15, codes >> 4), -1).reshape(codes.shape[0], -1).long().cpu()
    e = scales.cpu().int()
    s = torch.where(e == 255, torch.tensor(math.nan, dtype=torch.float64), _pow2(e - 127))
    return E2M1[c] * s.repeat_interleave(32, 1)


def random_mx4(g, n, k, spread=6):
    codes = torch.randint(0, 256, (n, k // 2), generator=g, device=DEV, dtype=torch.uint8)
    scales = torch.randint(118 - spread, 118 + spread, (n, k // 32), generator=g, device=DEV).to(torch.uint8)
    return codes, scales


def random_mx8(g, rows, k):
    data = torch.randint(0, 256, (rows, k), generator=g, device=DEV).to(torch.uint8)
    data = torch.where((data & 127) == 127, data - 1, data).view(torch.float8_e4m3fn)
    return ops.MX8Rows(data, torch.randint(115, 124, (rows, k // 32), generator=g, device=DEV).to(torch.uint8))


def outliers(g, rows, width):
    x = torch.randn((rows, width), generator=g, device=DEV)
    x[:, ::97] *= 50
    return (x * torch.exp(torch.randn((rows, 1), generator=g, device=DEV))).to(BF16)


def norm_reference(x, w, eps, residual=None):
    h = x.double() if residual is None else (residual.float() + x.float()).to(BF16).double()
    return w.double() * (h * (1 / torch.sqrt((h * h).mean(-1, keepdim=True) + eps)))


def same_mx8(got, y):
    code, byte = mx8_reference(y)
    assert torch.equal(got.scales.cpu(), byte)
    assert torch.equal(got.data.view(torch.uint8).cpu(), code)


# ------------------------------------------------------------------------------------------ 8-bit rows
@pytest.mark.parametrize("add", [False, True])
@pytest.mark.parametrize("rows,hidden", [(1, 32), (1, 4096), (3, 96), (7, 2080), (333, 1056), (64, 5120), (5, 16384), (2, 8224)])
def test_rmsnorm_mx8(rows, hidden, add):
    g = _gen(rows * 7 + hidden + add)
    x, w = outliers(g, rows, hidden), (1 + 0.3 * torch.randn(hidden, generator=g, device=DEV)).to(BF16)
    r = outliers(g, rows, hidden) if add else None
    want_r = (r.float() + x.float()).to(BF16) if add else None
    y = norm_reference(x, w, 1e-5, r)
    same_mx8(ops.rmsnorm_mx8(x, w, 1e-5, residual=r), y)
    if add:
        assert torch.equal(r, want_r)


def test_rmsnorm_mx8_rows_of_zeros_tiny_huge_and_bad_values():
    x = torch.randn((8, 256), generator=_gen(1), device=DEV)
    x[0] = 0
    x[1] *= 1e-30
    x[2] *= 1e30
    x[3, 40] = math.inf
    x[4, 70] = math.nan
    x[5, 32:64] *= 1e-36
    x[6, 5] = 3e38
    x = x.to(BF16)
    w = torch.ones(256, device=DEV, dtype=BF16)
    w[200:210] = 0
    w[211] = 1e30
    y = norm_reference(x, w, 1e-6)
    got = ops.rmsnorm_mx8(x, w, 1e-6)
    same_mx8(got, y)
    assert got.scales[4].eq(255).all() and got.scales[3].eq(255).sum() == 1
    assert torch.isnan(ops.mx8_unpack(got)[4]).all()


@pytest.mark.parametrize("rows,width", [(1, 32), (1, 14336), (3, 96), (65, 2080), (9, 14368)])
def test_silu_mul_mx8(rows, width):
    g = _gen(rows + width)
    both = (3 * torch.randn((rows, 2 * width), generator=g, device=DEV)).to(BF16)
    gate, up = both[:, :width], both[:, width:]
    y = gate.double() / (1 + torch.exp(-gate.double())) * up.double()
    same_mx8(ops.silu_mul_mx8(gate, up), y)


def test_silu_mul_mx8_every_gate_value():
    """All 65,536 bf16 gates beside up-projections of several sizes; blocks of neighbouring gates."""

    gate = torch.arange(65536, device=DEV).to(torch.uint16).view(BF16).view(-1, 512)
    for up in (1.0, -0.337890625, 3.0e-20, 1.1e30):
        u = torch.full_like(gate, up)
        d = gate.double()
        y = d / (1 + torch.exp(-d)) * u.double()
        over = y.abs() > 448 * 2.0 ** 127  # past the largest scale: NaN
        y = torch.where(over, torch.full_like(y, math.nan), y)
        same_mx8(ops.silu_mul_mx8(gate, u), y)


def test_mx8_values_are_ties_to_even_and_scales_break_at_448():
    """RMSNorm of weight-selected values: eps makes the factor 1, so the weights themselves are quantized."""

    k = 32 * 16
    x = torch.ones((1, k), device=DEV, dtype=BF16)
    w = torch.linspace(-3, 3, k, device=DEV).to(BF16).view(16, 32)
    w[0, 0], w[1, 0], w[2, 0], w[3, 0] = 1.75, 1.7578125, 3.5, 3.515625
    w = w.reshape(-1).contiguous()
    same_mx8(ops.rmsnorm_mx8(x, w, 0.0), w.double()[None])


def test_strided_and_higher_dim_rows():
    g = _gen(3)
    big = outliers(g, 6, 1024)
    x = big[:, 256:512]
    w = torch.ones(256, device=DEV, dtype=BF16)
    out = ops.MX8Rows(torch.zeros((6, 512), dtype=torch.uint8, device=DEV).view(torch.float8_e4m3fn)[:, :256],
                      torch.zeros((6, 40), dtype=torch.uint8, device=DEV)[:, 3:11])
    assert ops.rmsnorm_mx8(x, w, 1e-5, out=out) is out
    same_mx8(out, norm_reference(x, w, 1e-5))
    x3 = big.view(2, 3, 1024)[..., :256]
    got = ops.rmsnorm_mx8(x3, w, 1e-5)
    assert got.shape == (2, 3, 256)
    same_mx8(got, norm_reference(x3, w, 1e-5))
    assert torch.equal(ops.mx8_unpack(out).cpu().double(), mx8_values(out).to(BF16).double())
    assert ops.mx8_unpack(ops.rmsnorm_mx8(x[:0], w, 1e-5)).shape == (0, 256)


# ------------------------------------------------------------------------------------------ 4-bit weights
@pytest.mark.parametrize("n,k", [(1, 32), (16, 512), (17, 544), (100, 96), (33, 1600)])
def test_mx4_pack_and_unpack(n, k):
    codes, scales = random_mx4(_gen(n + k), n, k, spread=100)
    got = ops.mx4_unpack(ops.mx4_pack(codes, scales))
    want = mx4_values(codes, scales)
    assert torch.equal(got.double().cpu(), want)


def test_mx4_scale_255_is_nan_and_0_is_the_smallest():
    codes, scales = random_mx4(_gen(1), 16, 128)
    scales[2, 1], scales[5, 0] = 255, 0
    w = ops.mx4_pack(codes, scales)
    got = ops.mx4_unpack(w).double().cpu()
    assert torch.isnan(got[2, 32:64]).all() and not torch.isnan(got[2, :32]).any()
    assert torch.equal(got[5], mx4_values(codes, scales)[5])
    for x in (torch.ones((3, 128), device=DEV, dtype=BF16), random_mx8(_gen(2), 3, 128)):
        y = ops.mx4_linear(x, w)
        assert torch.isnan(y[:, 2]).all() and torch.isfinite(y[:, [0, 1, 3, 4, 5]]).all()


@pytest.mark.parametrize("n,k", [(1, 32), (40, 512), (17, 1056)])
def test_mx4_quantize(n, k):
    g = _gen(n)
    w = (torch.randn((n, k), generator=g, device=DEV) * torch.exp(4 * torch.randn((n, 1), generator=g, device=DEV))).to(BF16)
    w[0, :32] = 0
    if k > 64:
        w[0, 32:64] = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5, 6] * 4, device=DEV, dtype=BF16)  # ties
        w[-1, 64:96] *= 1e-38  # below the normal range
    got = ops.mx4_unpack(ops.mx4_quantize(w)).double().cpu()
    b = w.double().cpu().view(n, -1, 32)
    amax = b.abs().amax(-1, keepdim=True)
    m, e = torch.frexp(amax)
    e = torch.where(amax > 0, (e - 3 + (m > 0.75).to(e.dtype)).clamp(min=-127), torch.zeros_like(e))
    v = torch.ldexp(b, -e)
    mids = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5], dtype=torch.float64)
    lo, hi = torch.bucketize(v.abs(), mids), torch.bucketize(v.abs(), mids, right=True)
    code = torch.where(lo % 2 == 0, lo, hi)
    want = torch.ldexp(E2M1[code] * torch.where(torch.signbit(v), -1.0, 1.0).double(), e).view(n, k)
    assert torch.equal(got, want)


def group_maxima(v):
    return v.abs().view(v.shape[0], -1, 8).amax(-1)


ROWS, TILES = 1, 2


@pytest.fixture(params=[ROWS, TILES], ids=["rows", "tiles"])
def kernel(request, monkeypatch):
    """Every product of the test on this kernel (the Python body makes the calls)."""

    class Args(_lib.Mx4LinearArgs):
        def __init__(self):
            super().__init__()
            self.kernel = request.param

    monkeypatch.setattr(_lib, "Mx4LinearArgs", Args)
    monkeypatch.setattr(ops, "_host", None)
    monkeypatch.setattr(ops, "_host_bound", False)
    return request.param


def check_linear(x, xv, codes, scales, bias=None, out=None):
    w = ops.mx4_pack(codes, scales)
    got = ops.mx4_linear(x, w, bias=bias, out=out)
    wv = mx4_values(codes, scales).to(DEV)
    xv = xv.to(DEV)
    want = xv @ wv.t()
    mag = xv.abs() @ wv.abs().t()
    if bias is not None:
        want, mag = want + bias.double(), mag + bias.double().abs()
    tol = 2.0 ** -8 * want.abs() + (codes.shape[1] * 2 + 16) * 2.0 ** -24 * mag
    if isinstance(x, ops.MX8Rows):
        tol = tol + 7 * 2.0 ** -13 * (group_maxima(xv) @ group_maxima(wv).t())
    err = (got.double() - want).abs()
    assert bool((err <= tol).all()), float((err / tol.clamp(min=1e-300)).max())
    return got


SHAPES = [(1, 1, 32), (1, 16, 512), (1, 4096, 4096), (1, 2050, 14336), (2, 100, 96), (7, 33, 544), (15, 48, 1568), (16, 6144, 512),
          (17, 250, 1024), (31, 1000, 160), (32, 4096, 2048), (33, 17, 4064), (48, 8192, 320), (50, 130, 128), (64, 16400, 256),
          (65, 129, 288), (100, 1000, 1056), (128, 256, 512), (129, 384, 640), (250, 300, 96), (257, 513, 2080),
          (512, 512, 512), (1000, 6144, 1024), (1001, 6161, 416), (3000, 2060, 96)]


@pytest.mark.parametrize("m,n,k", SHAPES)
def test_linear_bf16_rows(m, n, k, kernel):
    g = _gen(m + n + k)
    codes, scales = random_mx4(g, n, k)
    x = outliers(g, m, k)
    bias = torch.randn(n, generator=g, device=DEV).to(BF16) if n % 2 else None
    check_linear(x, x.double(), codes, scales, bias)


@pytest.mark.parametrize("m,n,k", SHAPES)
def test_linear_mx8_rows(m, n, k, kernel):
    g = _gen(m + n + k + 1)
    codes, scales = random_mx4(g, n, k)
    x = random_mx8(g, m, k)
    bias = torch.randn(n, generator=g, device=DEV).to(BF16) if n % 2 else None
    check_linear(x, mx8_values(x), codes, scales, bias)


@pytest.mark.parametrize("m", [1, 300])
def test_mx8_products_that_cancel(m, kernel):
    """256 - 256 + 2^-b: the row kernel's products are exact; the tile kernel keeps 2^-5 and more among eight columns
    and any size in another eight."""

    w = ops.mx4_pack(torch.full((16, 256), 0x22, dtype=torch.uint8, device=DEV),
                     torch.full((16, 16), 127, dtype=torch.uint8, device=DEV))
    for at in (2, 7, 8, 31, 40, 300):
        for b in (5, 6, 9):
            x = torch.zeros((m, 512), dtype=torch.float32, device=DEV)
            x[:, 0], x[:, 1], x[:, at] = 256, -256, 2.0 ** -b
            x = ops.MX8Rows(x.to(torch.float8_e4m3fn), torch.full((m, 16), 127, dtype=torch.uint8, device=DEV))
            want = 0.0 if kernel == TILES and at < 8 and b > 5 else 2.0 ** -b
            assert ops.mx4_linear(x, w).eq(want).all(), (at, b)


@pytest.mark.parametrize("m,n,mx8", [(96, 28672, False), (96, 28672, True), (1000, 6144, True), (1000, 6144, False),
                                     (64, 28672, False), (32, 28672, False), (16, 28672, True), (17, 28672, True)])
def test_linear_kernels_chosen_by_size(m, n, mx8):
    """Without a fixed kernel the call equals the one whose sizes choose it."""

    g = _gen(m)
    w = ops.mx4_pack(*random_mx4(g, n, 256))
    x = random_mx8(g, m, 256) if mx8 else outliers(g, m, 256)
    a = _lib.Mx4LinearArgs()
    out = torch.empty((m, n), device=DEV, dtype=BF16)
    a.struct_size, a.rows, a.out_features, a.in_features = ctypes.sizeof(a), m, n, 256
    a.kernel = TILES if m > (16 if mx8 else 32) else ROWS
    data = x.data if mx8 else x
    a.x, a.x_stride, a.x_format = data.data_ptr(), 256, int(mx8)
    if mx8:
        a.x_scales, a.x_scale_stride = x.scales.data_ptr(), 8
    a.weight, a.out, a.out_stride = w.data.data_ptr(), out.data_ptr(), n
    _lib.check(_lib.load().lkv_mx4_linear(ctypes.byref(a), torch.cuda.current_stream().cuda_stream), "lkv_mx4_linear")
    assert torch.equal(out, ops.mx4_linear(x, w))


@pytest.mark.parametrize("mx8", [False, True])
@pytest.mark.parametrize("m,n,k", [(1030, 8001, 544), (1030, 8001, 640), (129, 28700, 160), (129, 28700, 640), (129, 28700, 32), (300, 5000, 1152)])
def test_linear_large_tiles(m, n, k, mx8):
    """Sizes that fill the card with tiles: the largest of them, cut at both edges, with scales in whole words and not."""

    g = _gen(m + n + k)
    codes, scales = random_mx4(g, n, k)
    bias = torch.randn(n, generator=g, device=DEV).to(BF16) if n % 2 else None
    x = random_mx8(g, m, k) if mx8 else outliers(g, m, k)
    check_linear(x, mx8_values(x) if mx8 else x.double(), codes, scales, bias)


@pytest.mark.parametrize("m", [1, 5, 40, 300])
def test_linear_bad_values_stay_in_their_row(m, kernel):
    """An infinity or NaN in one row of x: that row is what the products say, every other row is as without it."""

    g = _gen(m)
    codes, scales = random_mx4(g, 48, 640)
    codes[0], codes[1] = 0x22, 0xAA  # rows of 1.0 and of -1.0
    x = torch.randn((m, 640), generator=g, device=DEV).to(BF16)
    w = ops.mx4_pack(codes, scales)
    clean = ops.mx4_linear(x, w)
    x2 = x.clone()
    x2[m // 2, 333] = math.inf
    y = ops.mx4_linear(x2, w)
    keep = [i for i in range(m) if i != m // 2]
    assert torch.equal(y[keep], clean[keep])
    assert y[m // 2, 0] == math.inf and y[m // 2, 1] == -math.inf
    x2[m // 2, 333] = math.nan
    y = ops.mx4_linear(x2, w)
    assert torch.equal(y[keep], clean[keep]) and torch.isnan(y[m // 2]).all()


@pytest.mark.parametrize("mx8", [False, True])
@pytest.mark.parametrize("m", [3, 20, 200])
def test_linear_strided_rows_and_untouched_neighbours(m, mx8, kernel):
    g = _gen(m)
    codes, scales = random_mx4(g, 70, 544)
    if mx8:
        whole = random_mx8(g, m, 1088)
        x = ops.MX8Rows(whole.data[:, 544:], whole.scales[:, 17:])
        values = mx8_values(x)
    else:
        x = outliers(g, m, 1088)[:, 544:]
        values = x.double()
    out = torch.full((m + 2, 101), 7.0, device=DEV, dtype=BF16)
    check_linear(x, values, codes, scales, out=out[1:-1, 5:75])
    assert out[0].eq(7).all() and out[-1].eq(7).all() and out[:, :5].eq(7).all() and out[:, 75:].eq(7).all()
    if not mx8:
        y = ops.mx4_linear(x.unflatten(0, (1, m)), ops.mx4_pack(codes, scales))
        assert y.shape == (1, m, 70) and torch.equal(y[0], out[1:-1, 5:75])


@pytest.mark.parametrize("mx8", [False, True])
@pytest.mark.parametrize("m,n,k", [(70001, 24, 64), (3, 40, 131104), (70, 17, 65568)])
def test_linear_many_rows_and_long_ones(m, n, k, mx8, kernel):
    g = _gen(m + k)
    codes, scales = random_mx4(g, n, k)
    x = random_mx8(g, m, k) if mx8 else outliers(g, m, k)
    check_linear(x, mx8_values(x) if mx8 else x.double(), codes, scales, None)


def test_offsets_past_32_bits(kernel):
    """Outputs and rows past 2^31 elements: the last rows are what they are by themselves."""

    g = _gen(15)
    codes, scales = random_mx4(g, 2064, 32)
    w = ops.mx4_pack(codes, scales)
    x = torch.randn((1 << 20, 32), generator=g, device=DEV).to(BF16)
    assert torch.equal(ops.mx4_linear(x, w)[-100:], ops.mx4_linear(x[-100:].clone(), w))
    q = ops.silu_mul_mx8(x, x)
    assert torch.equal(ops.mx4_linear(q, w)[-100:], ops.mx4_linear(ops.MX8Rows(q.data[-100:], q.scales[-100:]), w))
    n = torch.ones(4096, device=DEV, dtype=BF16)
    big = torch.randn((1 << 10, 4096), generator=g, device=DEV).to(BF16).repeat(530, 1)  # 2^31 and 50 million
    for op in (lambda t: ops.rmsnorm_mx8(t, n, 1e-5), lambda t: ops.silu_mul_mx8(t, t)):
        q = op(big)
        few = op(big[-100:].clone())
        assert torch.equal(q.scales[-100:], few.scales)
        assert torch.equal(q.data[-100:].view(torch.uint8), few.data.view(torch.uint8))
        assert torch.equal(ops.mx8_unpack(q)[-100:], ops.mx8_unpack(few))
        del q


@pytest.mark.parametrize("mx8", [False, True])
@pytest.mark.parametrize("m", [1, 20, 200])
def test_linear_nan_block_of_the_weight(m, mx8, kernel):
    """Scale byte 255 in one block: NaN in that output feature, the others as without it."""

    g = _gen(14)
    codes, scales = random_mx4(g, 40, 672)
    x = random_mx8(g, m, 672) if mx8 else outliers(g, m, 672)
    want = ops.mx4_linear(x, ops.mx4_pack(codes, scales))
    scales[13, 20] = 255
    got = ops.mx4_linear(x, ops.mx4_pack(codes, scales))
    assert torch.isnan(got[:, 13]).all()
    got[:, 13] = want[:, 13]
    assert torch.equal(got, want)


@pytest.mark.parametrize("mx8", [False, True])
def test_one_row_of_any_stride(mx8, kernel):
    """The first row of a matrix whose rows are not 16-byte multiples apart."""

    g = _gen(12)
    codes, scales = random_mx4(g, 40, 96)
    if mx8:
        whole = random_mx8(g, 3, 128)
        data = torch.zeros((3, 101), device=DEV, dtype=torch.uint8).view(torch.float8_e4m3fn)
        data[:1, :96].view(torch.uint8).copy_(whole.data[:1, :96].view(torch.uint8))
        x = ops.MX8Rows(data[:1, :96], whole.scales[:1, :3])
        values = mx8_values(ops.MX8Rows(whole.data[:1, :96].contiguous(), whole.scales[:1, :3].contiguous()))
    else:
        x = outliers(g, 3, 101)[:1, :96]
        values = x.double()
    check_linear(x, values, codes, scales, None)


def test_norm_onto_its_own_residual():
    """residual = x: the row is doubled in place, then normalised."""

    g = _gen(13)
    x, w = outliers(g, 9, 2080), (1 + 0.3 * torch.randn(2080, generator=g, device=DEV)).to(BF16)
    want = (x.float() + x.float()).to(BF16)
    y = norm_reference(x, w, 1e-5, x)
    same_mx8(ops.rmsnorm_mx8(x, w, 1e-5, residual=x), y)
    assert torch.equal(x, want)


@pytest.mark.parametrize("m", [5, 200])
def test_linear_past_the_rows_and_columns_reads_nothing_that_counts(m, kernel):
    """NaN beside the rows of x (the next columns of a wider tensor), and in every place of the columns' tile before, does
    not reach the product."""

    g = _gen(9)
    nan = torch.full((m, 512), math.nan, device=DEV, dtype=BF16)
    assert torch.isnan(ops.mx4_linear(nan, ops.mx4_pack(*random_mx4(g, 40, 512)))).all()
    codes, scales = random_mx4(g, 40, 160)
    wide = nan.clone()
    wide[:, :160] = torch.randn((m, 160), generator=g, device=DEV)
    check_linear(wide[:, :160], wide[:, :160].double(), codes, scales)
    x8 = random_mx8(g, m, 160)
    data = torch.full((m, 512), 127, device=DEV, dtype=torch.uint8)
    data[:, :160] = x8.data.view(torch.uint8)
    s = torch.full((m, 16), 255, device=DEV, dtype=torch.uint8)
    s[:, :5] = x8.scales
    x = ops.MX8Rows(data.view(torch.float8_e4m3fn)[:, :160], s[:, :5])
    check_linear(x, mx8_values(x8), codes, scales)


def test_linear_same_bits_every_time_and_for_every_row_count():
    """A row's result does not depend on the call's other data, and two runs give the same bits."""

    g = _gen(4)
    codes, scales = random_mx4(g, 300, 1024)
    w = ops.mx4_pack(codes, scales)
    x = outliers(g, 64, 1024)
    y = ops.mx4_linear(x, w)
    assert torch.equal(y, ops.mx4_linear(x, w))
    assert torch.equal(y[16:32], ops.mx4_linear(x[16:32].clone(), w))
    q = ops.rmsnorm_mx8(x, torch.ones(1024, device=DEV, dtype=BF16), 1e-5)  # few rows: the products of their values
    assert torch.equal(ops.mx4_linear(q, w), ops.mx4_linear(ops.mx8_unpack(q), w))


def test_empty_rows():
    codes, scales = random_mx4(_gen(0), 16, 64)
    assert ops.mx4_linear(torch.empty((0, 64), device=DEV, dtype=BF16), ops.mx4_pack(codes, scales)).shape == (0, 16)


def test_other_stream_and_graph_replays():
    """The layer's operators in a row on a side stream, captured and replayed with new inputs, against eager calls."""

    g = _gen(11)
    hidden, width, rows = 512, 1056, 6
    w1, w2 = ops.mx4_pack(*random_mx4(g, 2 * width, hidden)), ops.mx4_pack(*random_mx4(g, hidden, width))
    norm = torch.ones(hidden, device=DEV, dtype=BF16)

    def block(x, residual):
        h = ops.rmsnorm_mx8(x, norm, 1e-5, residual=residual)
        both = ops.mx4_linear(h, w1)
        return ops.mx4_linear(ops.silu_mul_mx8(both[:, :width], both[:, width:]), w2)

    x, r = outliers(g, rows, hidden), outliers(g, rows, hidden)
    r0 = r.clone()
    want = block(x, r)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        r.copy_(r0)
        got = block(x, r)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = block(x, r)
    for seed in range(3):
        x.copy_(outliers(_gen(100 + seed), rows, hidden))
        r.copy_(r0)
        graph.replay()
        got = captured.clone()
        r.copy_(r0)
        assert torch.equal(got, block(x, r))
        torch.cuda.synchronize()


def test_block_against_64_bits():
    """norm -> gate/up -> SwiGLU -> down as a decode step runs them, against the same steps in 64 bits with their
    8-bit and bf16 roundings: an intermediate bf16 that rounds the other way (fp32 sums against 64-bit ones) moves its
    8-bit value by at most one step, 2^-3 of it; at most 2 % of them do (1056-term fp32 sums stay within 2^-16 of
    their magnitude, 2^-8 of a bf16 step times the cancellation), so the result is within sqrt(0.02) * 2^-3 < 2 %."""

    g = _gen(12)
    hidden, width, rows = 1024, 1056, 9
    c1, s1 = random_mx4(g, 2 * width, hidden, spread=1)
    c2, s2 = random_mx4(g, hidden, width, spread=1)
    x, r = outliers(g, rows, hidden), outliers(g, rows, hidden)
    norm = (1 + 0.1 * torch.randn(hidden, generator=g, device=DEV)).to(BF16)
    y = norm_reference(x, norm, 1e-5, r)
    h = ops.rmsnorm_mx8(x, norm, 1e-5, residual=r)
    same_mx8(h, y)
    both = ops.mx4_linear(h, ops.mx4_pack(c1, s1))
    got = ops.mx4_linear(ops.silu_mul_mx8(both[:, :width], both[:, width:]), ops.mx4_pack(c2, s2))
    b = (mx8_values(h) @ mx4_values(c1, s1).t()).to(BF16).double()
    gate, up = b[:, :width], b[:, width:]
    code, byte = mx8_reference(gate / (1 + torch.exp(-gate)) * up)
    m = mx8_values(ops.MX8Rows(code.to(DEV).view(torch.float8_e4m3fn), byte.to(DEV)))
    want = m @ mx4_values(c2, s2).t()
    assert float((got.double().cpu() - want).norm() / want.norm()) < 0.02
