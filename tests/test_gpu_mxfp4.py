"""MXFP4 quantisation, dequantisation, scale layout and product on the GPU against
exact restatements of their definitions."""
import numpy as np
import pytest

import dragonwing_edge_rs_b200 as dw
from dragonwing_edge_rs_b200 import ops
from tests import _mxfp4_ref as R

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def be():
    with dw.CudaBackend(0) as b:
        yield b


def operand(be, codes, scales, k, fill=0xAB):
    """Device buffers of an operand; scale places past the last row hold `fill`."""
    return be.upload_array(R.pack_codes(codes)), be.upload_array(R.pack_scales(scales, k, fill))


def run_quantize(be, raw, dtype, rows, k, pitch=0):
    x = be.upload_array(raw)
    q = be.upload_array(np.full(ops.mxfp4_code_bytes(rows, k), 0xCD, np.uint8))
    s = be.upload_array(np.full(ops.mxfp4_scale_bytes(rows, k), 0xAB, np.uint8))
    ops.quantize_mxfp4(be, x, R.DTYPES[dtype], rows, k, q, s, pitch)
    return be.download_array(q, np.uint8), be.download_array(s, np.uint8)


def check_quantized(q, s, x, k):
    rows = x.shape[0]
    codes, scales = R.quantize(x)
    got = R.unpack_codes(q, rows, k)
    np.testing.assert_array_equal(s, R.pack_scales(scales, k, 0xAB))  # rows past the last: left as they were
    bad = np.repeat(scales == 255, 32, 1)
    np.testing.assert_array_equal(np.where(bad, 0, got), np.where(bad, 0, codes))
    assert not got[bad].any()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,k,gap", [(1, 1, 0), (1, 4096, 0), (3, 31, 0), (2, 32, 0), (129, 33, 3), (257, 130, 0),
                                        (31, 1010, 15), (5, 11008, 0), (1000, 97, 8), (2, 40000, 0)])
def test_quantize(be, dtype, rows, k, gap):
    rng = np.random.default_rng(rows * 1000 + k)
    wide = rng.normal(0, 1, (rows, k + gap)) * np.exp(rng.normal(0, 2, (rows, k + gap)))
    wide[rng.random(wide.shape) < 0.05] = 0
    raw, val = R.to_type(wide, dtype)
    q, s = run_quantize(be, raw.reshape(-1)[:(rows - 1) * (k + gap) + k], dtype, rows, k, k + gap if gap else 0)
    check_quantized(q, s, val[:, :k], k)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("start", [0, 1, 2, 3, 4, 8])
@pytest.mark.parametrize("gap", [0, 1, 2, 4])
def test_quantize_starts_anywhere(be, dtype, start, gap):
    """A slice that begins `start` elements into its buffer, every alignment of its rows; NaN around it."""
    rows, k = 133, 104
    rng = np.random.default_rng(start * 10 + gap)
    wide = np.full((rows, k + gap), np.nan)
    wide[:, :k] = rng.normal(0, 1, (rows, k))
    raw, val = R.to_type(wide, dtype)
    nan = R.to_type(np.full(start + 1, np.nan), dtype)[0]
    whole = be.upload_array(np.concatenate([nan[:start], raw.reshape(-1)[:rows * (k + gap) - gap], nan[:1]]))
    es = 4 if dtype == "f32" else 2
    x = be.wrap(whole.device_ptr + start * es, (rows * (k + gap) - gap) * es)
    q = be.upload_array(np.full(ops.mxfp4_code_bytes(rows, k), 0xCD, np.uint8))
    s = be.upload_array(np.full(ops.mxfp4_scale_bytes(rows, k), 0xAB, np.uint8))
    ops.quantize_mxfp4(be, x, R.DTYPES[dtype], rows, k, q, s, k + gap)
    check_quantized(be.download_array(q, np.uint8), be.download_array(s, np.uint8), val[:, :k], k)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("start", [1, 3, 4])
def test_dequantize_starts_anywhere(be, dtype, start):
    rows, k = 133, 104
    rng = np.random.default_rng(start)
    codes, scales = rng.integers(0, 16, (rows, 128)).astype(np.uint8), rng.integers(120, 134, (rows, 4)).astype(np.uint8)
    es = 4 if dtype == "f32" else 2
    whole = be.upload_array(np.full(rows * k + start + 5, 7, R.np_type(dtype)))
    q, s = operand(be, codes, scales, k)
    ops.dequantize_mxfp4(be, q, s, rows, k, be.wrap(whole.device_ptr + start * es, rows * k * es), R.DTYPES[dtype])
    raw = be.download_array(whole, R.np_type(dtype))
    assert (raw[:start] == 7).all() and (raw[start + rows * k:] == 7).all()
    got = R.from_type(raw[start:start + rows * k].copy(), dtype).reshape(rows, k)
    np.testing.assert_array_equal(got, R.to_type(R.values(codes, scales, k), dtype)[1])


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_quantize_ties_and_limits(be, dtype):
    """Every tie at several scales, powers of two and their neighbours, zeros of both signs, the type's
    smallest and largest values."""
    ties = [0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.0, 7.5, 4.0, 6.0, 0.0, -0.0]
    rows = []
    for e in (-20, -3, 0, 5, 12):
        for top in (4.0, 6.0, 7.5):
            v = [top] + ties + [-t for t in ties]
            rows.append((np.array(v + [0.0] * (32 - len(v))) if len(v) <= 32 else np.array(v[:32])) * 2.0 ** e)
    f = {"f32": (2.0 ** -149, 3.4028234e38), "f16": (2.0 ** -24, 65504.0), "bf16": (2.0 ** -133, 3.3895314e38)}[dtype]
    for lim in f:
        rows.append(np.full(32, lim))
        rows.append(np.concatenate([[lim], np.zeros(31)]))
        rows.append(np.concatenate([[-lim, lim * 0.5, lim * 0.25], np.full(29, -0.0)]))
    rows.append(np.zeros(32))
    raw, val = R.to_type(np.stack(rows), dtype)
    q, s = run_quantize(be, raw, dtype, len(rows), 32)
    check_quantized(q, s, val, 32)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_quantize_not_finite(be, dtype):
    """A block with a NaN or an infinity becomes NaN; its neighbours in the row do not."""
    x = np.tile(np.linspace(-3, 3, 100), (4, 1))
    x[0, 5], x[1, 40], x[2, 99], x[3, 31] = np.nan, np.inf, -np.inf, np.nan
    raw, val = R.to_type(x, dtype)
    q, s = run_quantize(be, raw, dtype, 4, 100)
    check_quantized(q, s, val, 100)
    qd, sd = be.upload_array(q), be.upload_array(s)
    y = be.alloc(4 * 100 * 4)
    ops.dequantize_mxfp4(be, qd, sd, 4, 100, y, ops.F32)
    got = be.download_array(y, np.float32).reshape(4, 100)
    want = R.values(*R.quantize(val), 100)
    np.testing.assert_array_equal(np.isnan(got), np.isnan(want))
    assert np.isnan(got[0, :32]).all() and np.isfinite(got[0, 32:]).all() and np.isnan(got[2, 96:]).all()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,k", [(256, 512), (1, 1), (3, 33), (129, 130), (2, 40000)])
def test_dequantize(be, dtype, rows, k):
    """Every scale byte and code: exact where the type holds the value, else rounded once."""
    rng = np.random.default_rng(k)
    nb = R.blocks(k)
    codes = rng.integers(0, 16, (rows, nb * 32)).astype(np.uint8)
    scales = (np.arange(rows * nb) % 256).reshape(rows, nb).astype(np.uint8)
    q, s = operand(be, codes, scales, k)
    y = be.alloc(rows * k * (4 if dtype == "f32" else 2))
    ops.dequantize_mxfp4(be, q, s, rows, k, y, R.DTYPES[dtype])
    got = R.from_type(be.download_array(y, np_raw(dtype)), dtype).reshape(rows, k)
    with np.errstate(over="ignore"):
        want = R.to_type(R.values(codes, scales, k), dtype)[1]
    np.testing.assert_array_equal(got, want)


def np_raw(dtype):
    return R.np_type(dtype)


@pytest.mark.parametrize("rows,k", [(1, 1), (128, 128), (130, 4100), (7, 64)])
def test_pack_scales(be, rows, k):
    sc = np.random.default_rng(k).integers(0, 256, (rows, R.blocks(k))).astype(np.uint8)
    s = be.upload_array(np.full(ops.mxfp4_scale_bytes(rows, k), 0xAB, np.uint8))
    ops.pack_scales_mxfp4(be, be.upload_array(sc), rows, k, s)
    np.testing.assert_array_equal(be.download_array(s, np.uint8), R.pack_scales(sc, k, 0xAB))


# ---------------------------------------------------------------------------
# the product
# ---------------------------------------------------------------------------

def random_operand(rng, rows, k, lo=127, hi=128):
    """Random codes with scale exponents lo..hi - 127 and zero codes past k."""
    nb = R.blocks(k)
    codes = rng.integers(0, 16, (rows, nb * 32)).astype(np.uint8)
    codes[:, k:] = 0
    return codes, rng.integers(lo, hi + 1, (rows, nb)).astype(np.uint8)


def run_gemm(be, a, b, m, n, k, dtype="f32", bias=None, act=0):
    y = be.upload_array(np.full(m * n * (4 if dtype == "f32" else 2), 0x5A, np.uint8))
    ops.gemm_mxfp4(be, *a, *b, be.upload_array(bias) if bias is not None else None, y, R.DTYPES[dtype], m, n, k, act)
    return R.from_type(be.download_array(y, np_raw(dtype)), dtype).reshape(m, n)


SIZES = [(1, 1, 1), (1, 128, 32), (128, 128, 128), (128, 128, 64), (2, 3, 31), (129, 257, 257), (64, 96, 576), (16, 100, 40),
         (300, 130, 1000), (1, 4096, 4096), (7, 1000, 2056), (33, 640, 4128), (256, 384, 11008), (513, 1025, 96),
         (1100, 2100, 300), (100, 130, 64), (100, 1000, 2056), (128, 4096, 4128), (200, 300, 8200), (5100, 3890, 160)]


@pytest.mark.parametrize("m,n,k", SIZES)
def test_gemm_exact(be, m, n, k):
    """Codes with scales 1 and 2: products are multiples of 1/4 and every partial sum stays below 2^22, so
    f32 holds each of them exactly and the result is the exact one in any order of summation."""
    rng = np.random.default_rng(m + n + k)
    ac, asc = random_operand(rng, m, k)
    bc, bsc = random_operand(rng, n, k)
    A, B = R.values(ac, asc, k), R.values(bc, bsc, k)
    assert (np.abs(A) @ np.abs(B).T).max() < 2 ** 22
    got = run_gemm(be, operand(be, ac, asc, k), operand(be, bc, bsc, k), m, n, k)
    np.testing.assert_array_equal(got, A @ B.T)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("m,n,k,act,bias", [(1, 1000, 4096, 3, False), (37, 1000, 2056, 1, True), (130, 257, 999, 3, True),
                                            (256, 512, 11008, 0, True), (5, 33, 70, 0, False),
                                            (5100, 3890, 96, 3, True), (5100, 3904, 96, 1, True), (64, 1003, 4200, 0, True),
                                            (100, 1004, 4200, 3, True), (300, 2052, 520, 3, True)])
def test_gemm_scales_bias_act(be, dtype, m, n, k, act, bias):
    """Scales over 2^+-6.  Products are exact; f32 sums in groups of at least 16 products: (k / 16 + 2)
    additions, each off by at most one step (2^-23, truncation included) of a partial sum, which sum |ab|
    bounds.  The bias addition rounds once more, silu (slope at most 1.1) adds 2^-24 times 8 + |v|, the
    store half a step of the type."""
    rng = np.random.default_rng(m * n + k)
    ac, asc = random_operand(rng, m, k, 121, 133)
    bc, bsc = random_operand(rng, n, k, 110, 116)
    A, B = R.values(ac, asc, k), R.values(bc, bsc, k)
    bv = rng.normal(0, 1, n).astype(np.float32) if bias else None
    got = run_gemm(be, operand(be, ac, asc, k), operand(be, bc, bsc, k), m, n, k, dtype, bv, act)
    v = A @ B.T + (bv if bias else 0)
    want = R.act(v, act)
    tol = 1.1 * ((k / 16 + 2) * 2.0 ** -23 * (np.abs(A) @ np.abs(B).T) + 2.0 ** -24 * np.abs(v))
    if act == 3:
        tol += 2.0 ** -24 * (8 + np.abs(v)) * np.abs(want)
    tol = tol * (1 + 2 * R.EPS[dtype]) + R.EPS[dtype] * np.abs(want) + 2.0 ** -25
    assert (np.abs(got - want) <= tol).all(), np.max(np.abs(got - want) / tol)


@pytest.mark.parametrize("m,n,k,act", [(1, 32, 32, 0), (1, 1000, 4096, 3), (5, 97, 300, 0), (37, 1000, 2056, 1), (130, 257, 999, 3),
                                       (300, 640, 512, 3), (5100, 3890, 96, 0), (256, 500, 11008, 3), (100, 1000, 2056, 0),
                                       (64, 1003, 96, 3)])
def test_gemm_to_mxfp4_is_quantized_gemm(be, m, n, k, act):
    rng = np.random.default_rng(m * n + k)
    a = operand(be, *random_operand(rng, m, k, 121, 133), k)
    b = operand(be, *random_operand(rng, n, k, 110, 116), k)
    bias = rng.normal(0, 1, n).astype(np.float32)
    y = run_gemm(be, a, b, m, n, k, "f32", bias, act)
    q, s = run_to(be, a, b, m, n, k, bias, act)
    check_quantized(q, s, y, n)


def run_to(be, a, b, m, n, k, bias, act):
    q = be.upload_array(np.full(ops.mxfp4_code_bytes(m, n), 0xCD, np.uint8))
    s = be.upload_array(np.full(ops.mxfp4_scale_bytes(m, n), 0xAB, np.uint8))
    ops.gemm_to_mxfp4(be, *a, *b, be.upload_array(bias) if bias is not None else None, q, s, m, n, k, act)
    return be.download_array(q, np.uint8), be.download_array(s, np.uint8)


@pytest.mark.parametrize("m,n,k", [(3, 40, 100), (200, 300, 520)])
def test_gemm_nan_stays_in_its_row_and_column(be, m, n, k):
    """A NaN block of A spoils its row, one of B its column, and the scale bytes past the last row (NaN here)
    nothing."""
    rng = np.random.default_rng(3)
    ac, asc = random_operand(rng, m, k)
    bc, bsc = random_operand(rng, n, k)
    asc[1, 2], bsc[7, 0] = 255, 255
    got = run_gemm(be, operand(be, ac, asc, k, 0xFF), operand(be, bc, bsc, k, 0xFF), m, n, k)
    nan = np.zeros((m, n), bool)
    nan[1], nan[:, 7] = True, True
    np.testing.assert_array_equal(np.isnan(got), nan)
    want = R.values(ac, asc, k) @ R.values(bc, bsc, k).T
    np.testing.assert_array_equal(got[~nan], want[~nan])


@pytest.mark.parametrize("m", [1, 5, 160])
def test_gemm_repeats_captured_and_eager(be, m):
    """The same bits on every call and on graph replay, beside another call on a second stream."""
    import ctypes
    from dragonwing_edge_rs_b200 import _lib as L
    n, k = 1000, 2056
    rng = np.random.default_rng(9)
    a = operand(be, *random_operand(rng, m, k, 121, 133), k)
    b = operand(be, *random_operand(rng, n, k, 110, 116), k)
    first = run_gemm(be, a, b, m, n, k)
    y = be.upload_array(np.zeros(m * n, np.float32))
    lib, g = L.load(), ctypes.c_void_p()
    be.synchronize(10000)
    with dw.CudaBackend(0) as other:
        y2 = other.alloc(m * n * 4)
        be._check(lib.dw_capture_begin(be.handle))
        ops.gemm_mxfp4(be, *a, *b, None, y, ops.F32, m, n, k)
        be._check(lib.dw_capture_end(be.handle, ctypes.byref(g)))
        for _ in range(20):
            be._check(lib.dw_graph_launch(be.handle, g))
            ops.gemm_mxfp4(other, *a, *b, None, y2, ops.F32, m, n, k)
        got, got2 = be.download_array(y, np.float32), other.download_array(y2, np.float32)
        lib.dw_graph_destroy(g)
        y2.free()
    np.testing.assert_array_equal(got.reshape(m, n).astype(np.float64), first)
    np.testing.assert_array_equal(got2, got)


def test_refusals(be):
    """Bad arguments are refused before any launch, with a reason."""
    from dragonwing_edge_rs_b200 import _lib as L
    m, n, k = 4, 8, 64
    x = be.alloc(m * k * 4)
    q, s = be.alloc(ops.mxfp4_code_bytes(m, k)), be.alloc(ops.mxfp4_scale_bytes(m, k))
    bq, bs = be.alloc(ops.mxfp4_code_bytes(n, k)), be.alloc(ops.mxfp4_scale_bytes(n, k))
    y, yq, ys = be.alloc(m * n * 4), be.alloc(ops.mxfp4_code_bytes(m, n)), be.alloc(ops.mxfp4_scale_bytes(m, n))
    odd = be.wrap(q.device_ptr + 1, q.len_bytes())
    before = be.launch_count()

    def refused(status, f, *a):
        with pytest.raises(dw.BackendError) as e:
            f(be, *a)
        assert e.value.status == status and e.value.message

    inv, size = L.DW_ERR_INVALID_ARG, L.DW_ERR_SIZE_MISMATCH
    refused(inv, ops.quantize_mxfp4, x, ops.F32, 0, k, q, s)
    refused(inv, ops.quantize_mxfp4, x, ops.F32, m, 0, q, s)
    refused(inv, ops.quantize_mxfp4, x, 7, m, k, q, s)
    refused(inv, ops.quantize_mxfp4, x, ops.F32, m, k, None, s)
    refused(inv, ops.quantize_mxfp4, None, ops.F32, m, k, q, s)
    refused(inv, ops.quantize_mxfp4, x, ops.F32, m, k, q, s, k - 1)
    refused(inv, ops.quantize_mxfp4, x, ops.F32, m, k, odd, s)
    refused(inv, ops.quantize_mxfp4, x, ops.F32, 1 << 62, k, q, s)
    refused(size, ops.quantize_mxfp4, x, ops.F16, m, k, q, s)
    refused(size, ops.quantize_mxfp4, x, ops.F32, m, k, q, s, k + 1)
    refused(size, ops.quantize_mxfp4, x, ops.F32, m, k, bq, s)
    refused(size, ops.dequantize_mxfp4, q, s, m, k, y, ops.F32)
    refused(inv, ops.dequantize_mxfp4, q, s, m, k, x, 3)
    refused(size, ops.pack_scales_mxfp4, x, m, k, s)
    refused(size, ops.gemm_mxfp4, q, s, bq, bs, None, y, ops.F16, m, n, k)
    refused(size, ops.gemm_mxfp4, q, s, q, s, None, y, ops.F32, m, n, k)
    refused(size, ops.gemm_mxfp4, q, s, bq, bs, y, y, ops.F32, m, n, k)
    refused(inv, ops.gemm_mxfp4, q, s, bq, bs, None, y, ops.F32, m, n, k, ops.EPI_RELU6)
    refused(inv, ops.gemm_mxfp4, q, s, bq, bs, None, None, ops.F32, m, n, k)
    refused(inv, ops.gemm_mxfp4, q, s, bq, bs, None, y, ops.F32, m, n, 0)
    refused(inv, ops.gemm_to_mxfp4, q, s, bq, bs, None, yq, None, m, n, k)
    refused(size, ops.gemm_to_mxfp4, q, s, bq, bs, None, q, ys, m, n, k)
    assert be.launch_count() == before
