"""Which kernel a call of mx4_linear takes, on both sides of every border of the rule.

2,080 columns make the row kernel's waves and the tile kernel add in different orders, so that their outputs
differ somewhere and an equal output names the kernel.  (Above 16 row tiles a CU one wave of the row kernel walks all
columns, in the tile kernel's order: such a call's bits say nothing.)"""

from __future__ import annotations

import ctypes

import pytest
import torch

from lastkv_amd import _lib, ops

from test_gpu_mx import _gen, outliers, random_mx4, random_mx8

pytestmark = pytest.mark.gpu
DEV = "cuda"
K = 2080
ROWS, TILES = 1, 2


def forced(x, w, kernel):
    mx8 = isinstance(x, ops.MX8Rows)
    data, n = x.data if mx8 else x, w.out_features
    out = torch.empty((data.shape[0], n), device=DEV, dtype=torch.bfloat16)
    a = _lib.Mx4LinearArgs()
    a.struct_size, a.rows, a.out_features, a.in_features, a.kernel = ctypes.sizeof(a), data.shape[0], n, K, kernel
    a.x, a.x_stride, a.x_format = data.data_ptr(), K, int(mx8)
    if mx8:
        a.x_scales, a.x_scale_stride = x.scales.data_ptr(), K // 32
    a.weight, a.out, a.out_stride = w.data.data_ptr(), out.data_ptr(), n
    _lib.check(_lib.load().lkv_mx4_linear(ctypes.byref(a), torch.cuda.current_stream().cuda_stream), "lkv_mx4_linear")
    return out


# (8-bit, rows, row tiles of the weight a CU, kernel): above 8 tiles of 16 x 32 a CU (8-bit rows 4), more than 32 rows (16)
@pytest.mark.parametrize("mx8,m,per_cu,extra,kernel", [
    (True, 128, 1, 0, ROWS), (True, 129, 1, 0, TILES), (True, 64, 2, 0, ROWS), (True, 64, 2, 1, TILES),
    (True, 16, 7, 0, ROWS), (True, 17, 7, 0, TILES), (True, 17, 4, 0, ROWS), (True, 17, 4, 1, TILES),
    (False, 256, 1, 0, ROWS), (False, 257, 1, 0, TILES), (False, 64, 4, 0, ROWS), (False, 64, 4, 1, TILES),
    (False, 32, 16, 0, ROWS), (False, 32, 17, 0, ROWS), (False, 33, 5, 0, TILES)])
def test_kernel_of_a_call(mx8, m, per_cu, extra, kernel):
    cus = torch.cuda.get_device_properties(0).multi_processor_count
    g = _gen(m + per_cu)
    w = ops.mx4_pack(*random_mx4(g, 16 * (cus * per_cu + extra), K))
    x = random_mx8(g, m, K) if mx8 else outliers(g, m, K)
    by_rows, by_tiles = forced(x, w, ROWS), forced(x, w, TILES)
    assert torch.equal(by_rows, by_tiles) == (per_cu > 16)
    assert torch.equal(ops.mx4_linear(x, w), by_rows if kernel == ROWS else by_tiles)
