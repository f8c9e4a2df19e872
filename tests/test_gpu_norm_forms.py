"""The norm without a residual: its quantised result into buffers of its own, and in place, for
every kernel."""
import numpy as np
import pytest

import dragonwing_edge_rs_b200 as dw
from dragonwing_edge_rs_b200 import ops
from tests import _mxfp4_ref as R

pytestmark = pytest.mark.gpu

# rows streamed by accesses of 8, 2 and 1 elements; rows in registers by the same; rows over 16384
CASES = [(400, 1024), (300, 8192), (297, 4094), (2401, 129), (300, 1001), (5, 1024), (6, 1010), (5, 333), (1, 7), (3, 20001)]


@pytest.fixture(scope="module")
def be():
    with dw.CudaBackend(0) as b:
        yield b


def inputs(be, rng, rows, c, pitch, dtype):
    raw, _ = R.to_type(rng.normal(0.5, 2, (rows, pitch)), dtype)
    raw = raw.reshape(-1)[:(rows - 1) * pitch + c]
    w, b = rng.normal(1, 0.3, c).astype(np.float32), rng.normal(0, 0.3, c).astype(np.float32)
    return raw, be.upload_array(w), be.upload_array(b)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("kind", [ops.NORM_RMS, ops.NORM_LAYER])
@pytest.mark.parametrize("rows,c", CASES)
def test_norm_to_mxfp4_is_quantised_norm(be, rows, c, kind, dtype):
    rng = np.random.default_rng(rows + c)
    raw, w, b = inputs(be, rng, rows, c, c, dtype)
    x = be.upload_array(raw)
    d = ops.NormDesc(rows, c, R.DTYPES[dtype], R.DTYPES[dtype], ops.F32, kind, eps=1e-6)
    y = be.alloc(rows * c * 4)
    ops.norm(be, d, x, w, b, y)
    codes, scales = R.quantize(be.download_array(y, np.float32).reshape(rows, c).astype(np.float64))
    q = be.upload_array(np.full(ops.mxfp4_code_bytes(rows, c), 0xCD, np.uint8))
    s = be.upload_array(np.full(ops.mxfp4_scale_bytes(rows, c), 0xAB, np.uint8))
    ops.norm_to_mxfp4(be, d, x, w, b, q, s)
    np.testing.assert_array_equal(R.unpack_codes(be.download_array(q, np.uint8), rows, c), codes)
    np.testing.assert_array_equal(be.download_array(s, np.uint8), R.pack_scales(scales, c, 0xAB))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("gap", [0, 8, 3])
@pytest.mark.parametrize("rows,c", CASES)
def test_norm_in_place(be, rows, c, gap, dtype):
    rng = np.random.default_rng(rows + c + gap)
    pitch = c + gap
    raw, w, b = inputs(be, rng, rows, c, pitch, dtype)
    x, other = be.upload_array(raw), be.upload_array(raw)  # what lies between the rows stays as it was
    t = R.DTYPES[dtype]
    d = ops.NormDesc(rows, c, t, t, t, ops.NORM_LAYER, eps=1e-6, x_pitch=pitch if gap else 0, y_pitch=pitch if gap else 0)
    ops.norm(be, d, x, w, b, other)
    want = be.download_array(other, R.np_type(dtype))
    ops.norm(be, d, x, w, b, x)
    np.testing.assert_array_equal(be.download_array(x, R.np_type(dtype)), want)
    if gap:
        pad = lambda v: np.concatenate([v, np.zeros(gap, v.dtype)]).reshape(rows, pitch)[:-1, c:]  # noqa: E731
        np.testing.assert_array_equal(pad(want), pad(raw))
