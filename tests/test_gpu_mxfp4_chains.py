"""Each MXFP4 operator right behind the one that writes what it reads, over buffers that earlier
calls have read with other contents: a kernel that starts while the one before it still runs must
read nothing before that one's writes."""
import numpy as np
import pytest

import dragonwing_edge_rs_b200 as dw
from dragonwing_edge_rs_b200 import ops
from tests import _mxfp4_ref as R
from tests.test_gpu_mxfp4 import random_operand

pytestmark = pytest.mark.gpu

STEPS = 24


@pytest.fixture(scope="module")
def be():
    with dw.CudaBackend(0) as b:
        yield b


@pytest.mark.parametrize("rows,k", [(1, 4096), (300, 1010), (2000, 512)])
def test_quantised_and_read_back(be, rows, k):
    """x0, x1, x0, ... through the same codes and scales."""
    rng = np.random.default_rng(k)
    xs = [R.to_type(rng.normal(0, s, (rows, k)), "bf16") for s in (1.0, 37.0)]
    bx = [be.upload_array(raw) for raw, _ in xs]
    q, s = be.alloc(ops.mxfp4_code_bytes(rows, k)), be.alloc(ops.mxfp4_scale_bytes(rows, k))
    ys = [be.alloc(rows * k * 4) for _ in range(STEPS)]
    for i, y in enumerate(ys):
        ops.quantize_mxfp4(be, bx[i % 2], ops.BF16, rows, k, q, s)
        ops.dequantize_mxfp4(be, q, s, rows, k, y, ops.F32)
    want = [R.values(*R.quantize(val), k) for _, val in xs]
    for i, y in enumerate(ys):
        np.testing.assert_array_equal(be.download_array(y, np.float32).reshape(rows, k), want[i % 2])


@pytest.mark.parametrize("m", [3, 200])
def test_product_of_what_was_just_written(be, m):
    """Scales by pack_scales, the bias by dequantize, then the product; whole numbers, so the result is exact."""
    n, k = 300, 520
    rng = np.random.default_rng(m)
    nb = R.blocks(k)
    a = random_operand(rng, m, k)
    bc = random_operand(rng, n, k)[0]
    aq, as_ = be.upload_array(R.pack_codes(a[0])), be.upload_array(R.pack_scales(a[1], k))
    bq = be.upload_array(R.pack_codes(bc))
    scales = [np.full((n, nb), v, np.uint8) for v in (127, 128)]
    bs_rows = [be.upload_array(v) for v in scales]
    bias = [random_operand(rng, 1, n) for _ in range(2)]
    bias_ops = [(be.upload_array(R.pack_codes(c)), be.upload_array(R.pack_scales(s, n))) for c, s in bias]
    bs, bb = be.alloc(ops.mxfp4_scale_bytes(n, k)), be.alloc(n * 4)
    ys = [be.alloc(m * n * 4) for _ in range(STEPS)]
    for i, y in enumerate(ys):
        ops.pack_scales_mxfp4(be, bs_rows[i % 2], n, k, bs)
        ops.dequantize_mxfp4(be, *bias_ops[i % 2], 1, n, bb, ops.F32)
        ops.gemm_mxfp4(be, aq, as_, bq, bs, bb, y, ops.F32, m, n, k)
    want = [R.values(*a, k) @ R.values(bc, scales[i], k).T + R.values(*bias[i], n) for i in range(2)]
    for i, y in enumerate(ys):
        np.testing.assert_array_equal(be.download_array(y, np.float32).reshape(m, n), want[i % 2])
