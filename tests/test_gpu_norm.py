"""Norms around a residual on the GPU against their float64 definitions."""
import numpy as np
import pytest

import dragonwing_edge_rs_b200 as dw
from dragonwing_edge_rs_b200 import ops
from tests import _mxfp4_ref as R

pytestmark = pytest.mark.gpu

NONE, RMS, LAYER = ops.NORM_NONE, ops.NORM_RMS, ops.NORM_LAYER


@pytest.fixture(scope="module")
def be():
    with dw.CudaBackend(0) as b:
        yield b


def norm_tol(x, kind, w, b, eps):
    """Bound of the f32 norm's error.  A thread adds at most t = max(32, c / 512) terms and the tree 10 more:
    a sum of squares is off by (t + 12) * 2^-24 relative, its root by half that, and rsqrt, the products by
    rstd and w and the addition of b round once each: (t / 2 + 10) * 2^-24 of |n w|.  A layer norm's mean is off
    by (t + 12) * 2^-24 * mean|x|, which shifts every element (and, to second order only, the variance), and
    x - mean rounds."""
    if kind == NONE:
        return np.zeros_like(x)
    u = 2.0 ** -24
    t = max(32, -(-x.shape[1] // 512))
    c = x - x.mean(-1, keepdims=True) if kind == LAYER else x
    r = 1 / np.sqrt((c * c).mean(-1, keepdims=True) + eps)
    wa = np.abs(w) if w is not None else 1.0
    tol = (t / 2 + 10) * u * np.abs(c) * r * wa
    if kind == LAYER:
        shift = (t + 12) * u * np.abs(x).mean(-1, keepdims=True)
        # the variance of the shifted elements gains shift^2, and 2 shift mean(c) = 0
        tol = tol + 1.01 * (shift + u * np.abs(c)) * r * wa + np.abs(c) * r * wa * (shift * r) ** 2
    return tol + (u * np.abs(R.norm(x, kind, w, b, eps)) if b is not None else 0)


def near(got, want, tol, dtype):
    tol = tol * (1 + R.EPS[dtype]) + R.EPS[dtype] * np.abs(want) + 2.0 ** -25
    bad = np.abs(got - want) > tol
    assert not bad.any(), (int(bad.sum()), float(np.max(np.abs(got - want) / tol)))


def pitched(v, dtype, pitch):
    """Rows `pitch` apart in a host array with NaN between them."""
    rows, c = v.shape
    raw, val = R.to_type(v, dtype)
    if pitch <= c:
        return raw, val
    out, _ = R.to_type(np.full((rows, pitch), np.nan), dtype)
    out[:, :c] = raw
    return out, val


CASES = [(1, 1), (1, 4096), (3, 7), (9, 32), (257, 64), (40, 101), (5, 1010), (6, 1024), (33, 576), (2, 5000), (3, 8192), (2, 11008),
         (2, 16383), (2, 16384), (3, 20001), (2, 40000),
         # many rows
         (333, 8), (300, 64), (1001, 104), (400, 1024), (297, 4096), (300, 8192), (299, 11008), (298, 16384),
         (300, 7), (301, 129), (500, 1001), (297, 4094), (299, 8191), (297, 11009), (296, 16383)]


@pytest.mark.parametrize("dtype,ydtype", [("f32", "f32"), ("f16", "f16"), ("bf16", "bf16"), ("bf16", "f32"), ("f32", "bf16")])
@pytest.mark.parametrize("kind", [RMS, LAYER])
@pytest.mark.parametrize("rows,c", CASES)
def test_norm(be, dtype, ydtype, kind, rows, c):
    rng = np.random.default_rng(rows + c)
    gap = rng.integers(0, 2) * 3
    raw, x = pitched(rng.normal(0.5, 1, (rows, c)) * np.exp(rng.normal(0, 1, (1, c))), dtype, c + gap)
    w, b = (rng.normal(1, 0.3, c).astype(np.float32), rng.normal(0, 0.3, c).astype(np.float32)) if rng.random() < 0.6 else (None, None)
    d = ops.NormDesc(rows, c, R.DTYPES[dtype], R.DTYPES[dtype], R.DTYPES[ydtype], kind, eps=1e-5, x_pitch=c + gap if gap else 0)
    y = be.alloc(rows * c * (4 if ydtype == "f32" else 2))
    up = lambda v: None if v is None else be.upload_array(v)  # noqa: E731
    ops.norm(be, d, be.upload_array(raw), up(w), up(b), y)
    got = R.from_type(be.download_array(y, R.np_type(ydtype)), ydtype).reshape(rows, c)
    near(got, R.norm(x, kind, w, b, 1e-5), norm_tol(x, kind, w, b, 1e-5), ydtype)


@pytest.mark.parametrize("dtype,res", [("f32", "f32"), ("f16", "f16"), ("bf16", "bf16"), ("bf16", "f32"), ("f16", "f32")])
@pytest.mark.parametrize("rows,c,post,pre,gate_rows", [(1, 4096, NONE, RMS, None), (7, 1010, RMS, RMS, 0), (10, 333, LAYER, LAYER, 4),
                                                       (70, 96, RMS, LAYER, 1), (3, 20001, LAYER, RMS, 2), (2, 16384, RMS, RMS, 0),
                                                       (5, 64, RMS, NONE, None), (300, 512, NONE, LAYER, 100),
                                                       (310, 4096, RMS, RMS, 0), (301, 2048, LAYER, LAYER, 100),
                                                       (305, 104, RMS, RMS, 1), (300, 5120, LAYER, RMS, 7),
                                                       (299, 11008, RMS, RMS, None), (1030, 72, RMS, NONE, 0), (298, 16384, RMS, RMS, 1),
                                                       (298, 8192, LAYER, RMS, 0), (600, 1024, RMS, LAYER, 3),
                                                       (333, 33, RMS, RMS, 1), (501, 1010, LAYER, LAYER, 250), (300, 4095, RMS, RMS, 7),
                                                       (297, 10003, NONE, RMS, 0), (700, 62, LAYER, RMS, None)])
def test_norm_residual(be, dtype, res, rows, c, post, pre, gate_rows):
    """`out` against float64, and y against the norm of the stored `out`."""
    rng = np.random.default_rng(rows * 7 + c)
    xr, x = R.to_type(rng.normal(0, 1, (rows, c)), dtype)
    rr, r = R.to_type(rng.normal(0, 2, (rows, c)), res)
    groups = 0 if gate_rows is None else -(-rows // gate_rows) if gate_rows else 1
    gr, g = R.to_type(rng.normal(0.5, 0.5, (groups, c)), dtype) if groups else (None, None)
    w0, w1 = rng.normal(1, 0.3, c).astype(np.float32), rng.normal(1, 0.3, c).astype(np.float32)
    b1 = rng.normal(0, 0.3, c).astype(np.float32)
    b0 = rng.normal(0, 0.3, c).astype(np.float32) if post == LAYER else None
    scale = 0.75
    d = ops.NormDesc(rows, c, R.DTYPES[dtype], R.DTYPES[res], R.DTYPES[dtype], pre, post, 1e-6, gate_rows or 0, scale)
    es, rs = (4 if dtype == "f32" else 2), (4 if res == "f32" else 2)
    out, y = be.alloc(rows * c * rs), be.alloc(rows * c * es)
    bx, bw0, bw1, bb1 = be.upload_array(xr), be.upload_array(w0), be.upload_array(w1), be.upload_array(b1)
    bg = be.upload_array(gr) if groups else None
    bb0 = be.upload_array(b0) if b0 is not None else None
    ops.norm_residual(be, d, bx, bw0, bb0, bg, be.upload_array(rr), out, bw1, bb1, y)
    raw_out = be.download_array(out, R.np_type(res))
    got = R.from_type(raw_out, res).reshape(rows, c)
    gv = g[np.arange(rows) // gate_rows if gate_rows else np.zeros(rows, int)] if groups else 1.0
    n = R.norm(x, post, w0, b0, 1e-6) * gv
    # the products by the gate and the scale, and the sum with the bias' part, round once each
    tol = scale * (np.abs(gv) * norm_tol(x, post, w0, b0, 1e-6) + 3 * 2.0 ** -24 * np.abs(n))
    if b0 is not None:
        tol = tol + 4 * 2.0 ** -24 * (np.abs(scale * gv * b0) + np.abs(r))
    near(got, r + scale * n, tol * 1.01, res)
    got_y = R.from_type(be.download_array(y, R.np_type(dtype)), dtype).reshape(rows, c)
    wy, by = (w1, b1) if pre != NONE else (None, None)
    near(got_y, R.norm(got, pre, wy, by, 1e-6), norm_tol(got, pre, wy, by, 1e-6), dtype)

    # in place, and without y: the same bits
    inplace = be.upload_array(rr)
    ops.norm_residual(be, d, bx, bw0, bb0, bg, inplace, inplace)
    np.testing.assert_array_equal(be.download_array(inplace, R.np_type(res)), raw_out)
    # the fused quantisation: what the quantiser makes of the f32 norm of `out`
    df = ops.NormDesc(rows, c, R.DTYPES[res], R.DTYPES[res], ops.F32, pre, eps=1e-6)
    yf = be.alloc(rows * c * 4)
    ops.norm(be, df, out, bw1, bb1, yf)
    q, s = (be.upload_array(np.full(f(rows, c), 0xAB, np.uint8)) for f in (ops.mxfp4_code_bytes, ops.mxfp4_scale_bytes))
    q2, s2 = (be.upload_array(np.full(f(rows, c), 0xAB, np.uint8)) for f in (ops.mxfp4_code_bytes, ops.mxfp4_scale_bytes))
    ops.quantize_mxfp4(be, yf, ops.F32, rows, c, q, s)
    out2 = be.alloc(rows * c * rs)
    ops.norm_residual_to_mxfp4(be, d, bx, bw0, bb0, bg, be.upload_array(rr), out2, bw1, bb1, q2, s2)
    np.testing.assert_array_equal(be.download_array(out2, R.np_type(res)), raw_out)
    np.testing.assert_array_equal(be.download_array(q2, np.uint8), be.download_array(q, np.uint8))
    np.testing.assert_array_equal(be.download_array(s2, np.uint8), be.download_array(s, np.uint8))
    ops.norm_to_mxfp4(be, df, out, bw1, bb1, q2, s2)
    np.testing.assert_array_equal(be.download_array(q2, np.uint8), be.download_array(q, np.uint8))
    np.testing.assert_array_equal(be.download_array(s2, np.uint8), be.download_array(s, np.uint8))


@pytest.mark.parametrize("dtype,res", [("f32", "f32"), ("bf16", "bf16"), ("f16", "f32")])
@pytest.mark.parametrize("rows,c,post,pre,gate_rows", [(2000, 4096, RMS, RMS, 0), (2001, 4096, NONE, RMS, None),
                                                       (149, 5120, RMS, RMS, 0), (901, 5128, LAYER, RMS, 1), (603, 6144, RMS, LAYER, 2),
                                                       (605, 6152, RMS, RMS, 0), (151, 7168, LAYER, RMS, 3), (603, 8192, RMS, RMS, 1),
                                                       (605, 8192, NONE, RMS, None), (152, 16384, NONE, RMS, None),
                                                       (905, 4098, RMS, RMS, 0), (904, 1021, LAYER, RMS, 2),
                                                       (40000, 64, NONE, RMS, None), (9000, 200, RMS, RMS, 0)])
def test_rows_that_pass_through_the_ring_more_than_once(be, dtype, res, rows, c, post, pre, gate_rows):
    test_norm_residual(be, dtype, res, rows, c, post, pre, gate_rows)


@pytest.mark.parametrize("rows", [9, 700])
@pytest.mark.parametrize("c", [200, 199])
def test_pitches(be, rows, c):
    """x, residual, out and y as slices of wider tensors: what lies between the rows is not touched."""
    rng = np.random.default_rng(2)
    xr, x = pitched(rng.normal(0, 1, (rows, c)), "f16", 208)
    rr, r = pitched(rng.normal(0, 1, (rows, c)), "f32", 211)
    d = ops.NormDesc(rows, c, ops.F16, ops.F32, ops.BF16, RMS, RMS, 1e-5, x_pitch=208, res_pitch=211, y_pitch=204)
    out = be.upload_array(np.full((rows, 211), 7, np.float32))
    y = be.upload_array(np.full((rows, 204), 0x4110, np.uint16))
    ops.norm_residual(be, d, be.upload_array(xr), None, None, None, be.upload_array(rr), out, None, None, y)
    got = be.download_array(out, np.float32, (rows, 211))
    assert (got[:, c:] == 7).all()
    near(got[:, :c].astype(np.float64), r + R.norm(x, RMS, None, None, 1e-5), norm_tol(x, RMS, None, None, 1e-5), "f32")
    yr = be.download_array(y, np.uint16, (rows, 204))
    assert (yr[:, c:] == 0x4110).all()
    g64 = got[:, :c].astype(np.float64)
    near(R.from_type(yr, "bf16")[:, :c], R.norm(g64, RMS, None, None, 1e-5), norm_tol(g64, RMS, None, None, 1e-5), "bf16")


@pytest.mark.parametrize("rows", [1, 5, 400])
@pytest.mark.parametrize("start", [1, 3, 8])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_tensors_that_start_anywhere(be, rows, start, dtype):
    """Tensors inside larger buffers, `start` elements in: the elements before and after them (NaN here, and
    closer than a 16-byte piece) are neither used nor changed."""
    c = 101
    rng = np.random.default_rng(start)
    es = 4 if dtype == "f32" else 2
    xr, x = R.to_type(rng.normal(0, 1, rows * c), dtype)
    rr, r = R.to_type(rng.normal(0, 1, rows * c), dtype)
    gr, g = R.to_type(rng.normal(0, 1, rows * c), dtype)
    nan = R.to_type(np.full(start, np.nan), dtype)[0]
    whole = [be.upload_array(np.concatenate([nan, v, nan[:1]])) for v in (xr, rr, gr, rr, xr)]
    bx, br, bg, bo, by = (be.wrap(b.device_ptr + start * es, rows * c * es) for b in whole)
    d = ops.NormDesc(rows, c, R.DTYPES[dtype], R.DTYPES[dtype], R.DTYPES[dtype], RMS, RMS, 1e-5, gate_rows=1)
    ops.norm_residual(be, d, bx, None, None, bg, br, bo, None, None, by)
    x, r, g = (v.reshape(rows, c) for v in (x, r, g))
    n = R.norm(x, RMS, None, None, 1e-5)
    raw = [be.download_array(b, R.np_type(dtype)) for b in whole]
    for b, v in zip(raw, (xr, rr, gr, None, None)):
        np.testing.assert_array_equal(b[:start], nan)
        np.testing.assert_array_equal(b[-1:], nan[:1])
        if v is not None:
            np.testing.assert_array_equal(b[start:-1], v)
    out = R.from_type(raw[3][start:-1].copy(), dtype).reshape(rows, c)
    near(out, r + g * n, 1.01 * np.abs(g) * (norm_tol(x, RMS, None, None, 1e-5) + 3 * 2.0 ** -24 * np.abs(n)), dtype)
    near(R.from_type(raw[4][start:-1].copy(), dtype).reshape(rows, c), R.norm(out, RMS, None, None, 1e-5),
         norm_tol(out, RMS, None, None, 1e-5), dtype)


@pytest.mark.parametrize("c", [100, 20001])
def test_constant_and_not_finite_rows(be, c):
    """A constant row (variance 0), a zero row, and NaN or infinity in one row leave the others alone."""
    x = np.random.default_rng(1).normal(0, 1, (5, c)).astype(np.float32)
    x[0], x[1], x[2, 3], x[3, 5] = 4.0, 0.0, np.nan, np.inf
    d = ops.NormDesc(5, c, ops.F32, ops.F32, ops.F32, LAYER, eps=1e-5)
    y = be.alloc(5 * c * 4)
    ops.norm(be, d, be.upload_array(x), None, None, y)
    got = be.download_array(y, np.float32, (5, c))
    assert (np.abs(got[:2]) <= 1e-3).all() and (got[1] == 0).all()
    assert np.isnan(got[2]).all() and np.isnan(got[3]).all()
    near(got[4:].astype(np.float64), R.norm(x[4:].astype(np.float64), LAYER, None, None, 1e-5),
         norm_tol(x[4:].astype(np.float64), LAYER, None, None, 1e-5), "f32")


def test_refusals(be):
    from dragonwing_edge_rs_b200 import _lib as L
    rows, c = 4, 64
    x, r, o, w = be.alloc(rows * c * 2), be.alloc(rows * c * 2), be.alloc(rows * c * 2), be.alloc(c * 4)
    big = be.alloc(rows * c * 4)
    ok = dict(rows=rows, c=c, x_dtype=ops.F16, res_dtype=ops.F16, y_dtype=ops.F16)
    before = be.launch_count()

    def refused(status, change, *a):
        with pytest.raises(dw.BackendError) as e:
            ops.norm_residual(be, ops.NormDesc(**{**ok, **change}), *a)
        assert e.value.status == status and e.value.message

    inv, size = L.DW_ERR_INVALID_ARG, L.DW_ERR_SIZE_MISMATCH
    good = (x, w, None, None, r, o)
    refused(inv, {"rows": 0}, *good)
    refused(inv, {"c": 0}, *good)
    refused(inv, {"x_dtype": 9}, *good)
    refused(inv, {"pre": 5}, *good)
    refused(inv, {"eps": -1.0}, *good)
    refused(inv, {"eps": float("nan")}, *good)
    refused(inv, {"res_scale": float("nan")}, *good)
    refused(inv, {"x_pitch": c - 1}, *good)
    refused(size, {"x_pitch": c + 1}, *good)
    refused(L.DW_ERR_UNSUPPORTED, {"x_dtype": ops.F32, "res_dtype": ops.F16}, big, w, None, None, r, o)
    refused(size, {"res_dtype": ops.F32}, *good)
    refused(size, {}, x, x, None, None, r, o)
    refused(size, {}, x, w, None, x, r, o)          # a gate of one row is wanted
    refused(size, {"gate_rows": 3}, x, w, None, x, r, o)
    refused(inv, {}, x, w, None, None, None, o)
    refused(inv, {}, x, w, None, None, r, None)
    refused(size, {}, x, w, None, None, r, o, None, None, w)
    with pytest.raises(dw.BackendError):
        ops.norm(be, ops.NormDesc(**ok), x, None, None, None)
    with pytest.raises(dw.BackendError):
        ops.norm_to_mxfp4(be, ops.NormDesc(**ok), x, None, None, x, w)
    assert be.launch_count() == before
