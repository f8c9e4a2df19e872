"""Products of few rows with so many outputs that the CTAs outnumber the SMs, and a K of one to
four blocks of 256: rings of one, two and three stages."""
import numpy as np
import pytest

import dragonwing_edge_rs_b200 as dw
from tests import _mxfp4_ref as R
from tests.test_gpu_mxfp4 import operand, random_operand, run_gemm

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("m,n,k", [(1, 32000, 256), (16, 20003, 300), (32, 28672, 512), (17, 19000, 700), (5, 40000, 1024), (1, 65536, 33)])
def test_exact(m, n, k):
    """Whole multiples of 1/4 below 2^22: exact in any order of summation."""
    rng = np.random.default_rng(m + n + k)
    ac, asc = random_operand(rng, m, k)
    bc, bsc = random_operand(rng, n, k)
    A, B = R.values(ac, asc, k), R.values(bc, bsc, k)
    assert (np.abs(A) @ np.abs(B).T).max() < 2 ** 22
    with dw.CudaBackend(0) as be:
        got = run_gemm(be, operand(be, ac, asc, k), operand(be, bc, bsc, k), m, n, k)
    np.testing.assert_array_equal(got, A @ B.T)
