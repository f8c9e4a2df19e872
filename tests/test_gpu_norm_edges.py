"""Norms of many rows whose tensors begin and end inside a 16-byte piece: the elements there come
into the ring by ordinary stores of several lanes, the others by bulk copies."""
import numpy as np
import pytest

import dragonwing_edge_rs_b200 as dw
from dragonwing_edge_rs_b200 import ops
from tests import _mxfp4_ref as R
from tests.test_gpu_norm import RMS, near, norm_tol

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def be():
    with dw.CudaBackend(0) as b:
        yield b


# 8 rows a step of the ring up to c = 512: the last step of 2401 rows has one row, whose bytes up to
# c = 3 all lie in the tensor's last piece (no bulk copy at all)
@pytest.mark.parametrize("start,gap", [(0, 3), (1, 0), (5, 3)])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,c", [(2401, 1), (2401, 3), (2403, 7), (2402, 30), (2401, 101), (700, 1001)])
def test_many_rows_that_start_anywhere(be, rows, c, dtype, start, gap):
    es = 4 if dtype == "f32" else 2
    pitch = c + gap
    n = (rows - 1) * pitch + c
    nan = R.to_type(np.full(start + 1, np.nan), dtype)[0]
    d = ops.NormDesc(rows, c, R.DTYPES[dtype], R.DTYPES[dtype], R.DTYPES[dtype], RMS, RMS, 1e-5, gate_rows=1,
                     x_pitch=pitch, res_pitch=pitch)
    for seed in range(3):
        rng = np.random.default_rng(rows * 100 + c + seed)

        def tensor(pitch):
            wide = np.full((rows, pitch), np.nan)
            wide[:, :c] = rng.normal(0, 1, (rows, c))
            raw, val = R.to_type(wide, dtype)
            raw = raw.reshape(-1)[:(rows - 1) * pitch + c]
            whole = be.upload_array(np.concatenate([nan[:start], raw, nan[:1]]))
            return whole, be.wrap(whole.device_ptr + start * es, raw.size * es), val[:, :c]

        (wx, bx, x), (wr, br, r), (wg, bg, g) = tensor(pitch), tensor(pitch), tensor(c)
        out, y = be.upload_array(np.full(n, 7, R.np_type(dtype))), be.alloc(rows * c * es)
        ops.norm_residual(be, d, bx, None, None, bg, br, out, None, None, y)
        raw = be.download_array(out, R.np_type(dtype))
        raw = np.concatenate([raw, np.full(gap, 7, raw.dtype)]).reshape(rows, pitch)
        assert (raw[:, c:] == 7).all()
        got = R.from_type(raw[:, :c], dtype).reshape(rows, c)
        v = R.norm(x, RMS, None, None, 1e-5)
        # one product by the gate, one sum
        near(got, r + g * v, 1.01 * np.abs(g) * (norm_tol(x, RMS, None, None, 1e-5) + 3 * 2.0 ** -24 * np.abs(v)), dtype)
        near(R.from_type(be.download_array(y, R.np_type(dtype)), dtype).reshape(rows, c), R.norm(got, RMS, None, None, 1e-5),
             norm_tol(got, RMS, None, None, 1e-5), dtype)
        # in place: the same bits
        ops.norm_residual(be, d, bx, None, None, bg, br, br)
        kept = be.download_array(wr, R.np_type(dtype))
        np.testing.assert_array_equal(kept[:start], nan[:start])
        np.testing.assert_array_equal(kept[start + n:], nan[:1])
        kept = np.concatenate([kept[start:start + n], np.full(gap, 7, raw.dtype)]).reshape(rows, pitch)[:, :c]
        np.testing.assert_array_equal(kept, raw[:, :c])
