"""NaN through the activations of the MXFP4 product: a block that is not finite makes its row or
column NaN, whatever the activation and the form of the result."""
import numpy as np
import pytest

import dragonwing_edge_rs_b200 as dw
from dragonwing_edge_rs_b200 import ops
from tests import _mxfp4_ref as R
from tests.test_gpu_mxfp4 import check_quantized, operand, random_operand, run_gemm, run_to

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def be():
    with dw.CudaBackend(0) as b:
        yield b


# few rows; pairs of CTAs; two pairs for one tile's K; 256 x 256 tiles
@pytest.mark.parametrize("m,n,k", [(3, 40, 100), (200, 300, 520), (200, 300, 8200), (5100, 3890, 96)])
@pytest.mark.parametrize("act", [ops.EPI_NONE, ops.EPI_RELU, ops.EPI_SILU])
def test_nan_passes_the_activation(be, m, n, k, act):
    rng = np.random.default_rng(m + act)
    ac, asc = random_operand(rng, m, k)
    bc, bsc = random_operand(rng, n, k)
    asc[1, 2], bsc[7, 0] = 255, 255
    nan = np.zeros((m, n), bool)
    nan[1], nan[:, 7] = True, True
    bias = np.zeros(n, np.float32)
    bias[9], bias[10], bias[11] = np.nan, np.inf, -np.inf
    nan[:, 9] = True
    nan[:, 11] |= act == ops.EPI_SILU  # -inf * 0
    a, b = operand(be, ac, asc, k), operand(be, bc, bsc, k)
    got = run_gemm(be, a, b, m, n, k, "f32", bias, act)
    np.testing.assert_array_equal(np.isnan(got), nan)
    inf = np.zeros((m, n), bool)
    inf[:, 10] = ~nan[:, 10]
    inf[:, 11] |= ~nan[:, 11] & (act == ops.EPI_NONE)
    np.testing.assert_array_equal(np.isinf(got), inf)
    if act == ops.EPI_RELU:
        assert (got[~nan] >= 0).all() and (got[~nan[:, 11], 11] == 0).all()
    check_quantized(*run_to(be, a, b, m, n, k, bias, act), got, n)  # scale byte 255 where a block has one
