"""The 4-bit operators where offsets pass 32 bits: sampled rows against their definitions."""
import numpy as np
import pytest
import torch

import dragonwing_edge_rs_b200 as dw
from dragonwing_edge_rs_b200 import ops
from tests import _mxfp4_ref as R
from tests.test_gpu_norm import near, norm_tol

pytestmark = pytest.mark.gpu

ROWS, C = 70000, 65536  # 4.59e9 elements
SAMPLE = [0, 1, 32767, 32768, 65535, 65536, 69999]


@pytest.fixture(scope="module")
def be():
    with dw.CudaBackend(0) as b:
        yield b


def wrap(be, t):
    return be.wrap(t.data_ptr(), t.numel() * t.element_size())


def rows_of(t, rows):
    return t[torch.tensor(rows, device=t.device)].float().cpu().numpy().astype(np.float64)


def test_quantize_and_back(be):
    x = torch.empty(ROWS, C, dtype=torch.bfloat16, device="cuda").normal_()
    q = torch.empty(ops.mxfp4_code_bytes(ROWS, C), dtype=torch.uint8, device="cuda")
    s = torch.empty(ops.mxfp4_scale_bytes(ROWS, C), dtype=torch.uint8, device="cuda")
    y = torch.empty_like(x)
    torch.cuda.synchronize()
    ops.quantize_mxfp4(be, wrap(be, x), ops.BF16, ROWS, C, wrap(be, q), wrap(be, s))
    ops.dequantize_mxfp4(be, wrap(be, q), wrap(be, s), ROWS, C, wrap(be, y), ops.BF16)
    be.synchronize(60000)
    np.testing.assert_array_equal(rows_of(y, SAMPLE), R.values(*R.quantize(rows_of(x, SAMPLE)), C))


def test_product(be):
    """y of 9.2 GB: products of +-1 and scales 1 are whole numbers below 2^8, exact in bf16."""
    k = 32
    rng = np.random.default_rng(1)
    ac = np.where(rng.random((ROWS, k)) < 0.5, 2, 10).astype(np.uint8)
    bc = np.where(rng.random((C, k)) < 0.5, 2, 10).astype(np.uint8)
    one = lambda rows: np.full((rows, 1), 127, np.uint8)  # noqa: E731
    a = be.upload_array(R.pack_codes(ac)), be.upload_array(R.pack_scales(one(ROWS), k))
    b = be.upload_array(R.pack_codes(bc)), be.upload_array(R.pack_scales(one(C), k))
    y = torch.empty(ROWS, C, dtype=torch.bfloat16, device="cuda")
    torch.cuda.synchronize()
    ops.gemm_mxfp4(be, *a, *b, None, wrap(be, y), ops.BF16, ROWS, C, k)
    be.synchronize(60000)
    A, B = R.values(ac[SAMPLE], one(len(SAMPLE)), k), R.values(bc, one(C), k)
    np.testing.assert_array_equal(rows_of(y, SAMPLE), A @ B.T)


@pytest.mark.parametrize("rows,c", [(1150000, 4095), (ROWS, C)])
def test_norm(be, rows, c):
    x = torch.empty(rows, c, dtype=torch.bfloat16, device="cuda").normal_()
    r = torch.empty_like(x).normal_()
    out, y = torch.empty_like(x), torch.empty_like(x)
    d = ops.NormDesc(rows, c, ops.BF16, ops.BF16, ops.BF16, ops.NORM_RMS, ops.NORM_RMS)
    torch.cuda.synchronize()
    ops.norm_residual(be, d, wrap(be, x), None, None, None, wrap(be, r), wrap(be, out), None, None, wrap(be, y))
    be.synchronize(60000)
    sample = [0, 1, 65536, rows // 2, rows - 2, rows - 1] if rows > ROWS else SAMPLE
    x64, r64, o64 = (rows_of(t, sample) for t in (x, r, out))
    n = R.norm(x64, 1, None, None, 1e-5)
    near(o64, r64 + n, 1.01 * (norm_tol(x64, 1, None, None, 1e-5) + 3 * 2.0 ** -24 * np.abs(n)), "bf16")
    near(rows_of(y, sample), R.norm(o64, 1, None, None, 1e-5), norm_tol(o64, 1, None, None, 1e-5), "bf16")
