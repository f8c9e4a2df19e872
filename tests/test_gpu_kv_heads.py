"""Head norms with the rotation, appending to the paged 8-bit cache and reading it back, against float64."""
import numpy as np
import pytest

import dragonwing_edge_rs_b200 as dw
from dragonwing_edge_rs_b200 import ops
from tests import _kv_ref as K
from tests import _mxfp4_ref as R

pytestmark = pytest.mark.gpu
HALF_STEP = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}


@pytest.fixture(scope="module")
def be():
    with dw.CudaBackend(0) as b:
        yield b


def values(raw, dtype):
    """The float64 values of downloaded bytes."""
    if dtype == "bf16":
        return (raw.view(np.uint16).astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    return raw.view(np.float32 if dtype == "f32" else np.float16).astype(np.float64)


def put(be, x, dtype):
    raw, val = R.to_type(np.ascontiguousarray(x), dtype)
    return be.upload_array(raw), np.asarray(val, np.float64)


def freqs(rot):
    return 10000.0 ** (-2.0 * np.arange(rot // 2) / max(rot, 1))


def rope_tolerance(x, kind, w, eps, want, rot, neighbours, dtype):
    """f32 arithmetic, in halves of its last place (2^-24): a sum of squares by chains of at most 16 and five levels
    is off by 21, a square root of its mean and reciprocal by 12 then, times a weight and a value 2 more; a turn's
    cosine and sine by 8 (the angle's own rounding is below 4), its products and sum 4 (all of the pair's size);
    a mean taken away is off by 23 of the mean of |x|."""
    y = K.norm(x, kind, w, eps)
    size = np.abs(y)
    if rot:
        i = np.arange(rot // 2)
        a, b = (2 * i, 2 * i + 1) if neighbours else (i, i + rot // 2)
        size = size.copy()
        size[..., a] = size[..., b] = size[..., a] + size[..., b]
    tol = 30 * 2.0 ** -24 * size
    if kind == 2:
        spread = np.abs(x).mean(-1, keepdims=True)
        std = np.sqrt(((x - x.mean(-1, keepdims=True)) ** 2).mean(-1, keepdims=True) + eps)
        tol = tol + 2 * 25 * 2.0 ** -24 * spread / std * (1.0 if w is None else np.abs(w).max())
    floor = {"f32": 1e-44, "f16": 2.0 ** -25, "bf16": 1e-40}[dtype]
    return tol * 1.01 + HALF_STEP[dtype] * (np.abs(want) + tol) + floor


CASES = [  # tokens, hq, hk, d, rot, neighbours, norm, offset, gap, far
    (1, 32, 8, 128, 128, False, 1, 0, 0, 0), (1, 1, 1, 64, 64, True, 0, 0, 0, 5), (7, 5, 2, 128, 64, False, 2, 8, 16, 1 << 20),
    (300, 3, 1, 64, 32, True, 1, 0, 0, 2000000000), (33, 2, 2, 96, 96, False, 1, 0, 8, 77), (5, 3, 1, 80, 20, False, 1, 3, 5, 9),
    (3, 2, 1, 512, 512, False, 1, 0, 0, 4), (9, 4, 2, 2, 2, False, 0, 1, 0, 100), (4, 2, 1, 250, 30, True, 2, 0, 0, 1000),
    (2000, 7, 3, 128, 0, False, 1, 0, 0, 0), (129, 1, 1, 16, 16, True, 1, 0, 0, 3)]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("case", CASES)
def test_norm_rope(be, dtype, case):
    n, hq, hk, d, rot, nb, kind, off, gap, far = case
    rng = np.random.default_rng(n + d)
    pitch = (hq + hk) * d + gap
    x, xv = put(be, rng.normal(0, 1, n * pitch + off) * np.exp(rng.normal(0, 1, n * pitch + off)), dtype)
    rows = np.lib.stride_tricks.as_strided(xv[off:], (n, pitch), (8 * pitch, 8)).copy()[:, :(hq + hk) * d].reshape(n, hq + hk, d)
    pos = (rng.integers(-far, far + 1, n) + (np.arange(n) if far < 1 << 30 else 0)).astype(np.int32)
    wq, wk = rng.normal(1, 0.3, (2, d)).astype(np.float32)
    es = 4 if dtype == "f32" else 2
    q_out = be.upload_array(np.full(n * hq * d * es, 0xAB, np.uint8))
    k_out = be.upload_array(np.full((n * hk * d + 3) * es, 0xAB, np.uint8))
    desc = ops.HeadDesc(hq, hk, d, rot, R.DTYPES[dtype], kind, 1e-5, nb)
    rope = ops.prepare_rope(be, freqs(rot)) if rot else None
    ops.norm_rope(be, desc, n, ops.Heads(x, off, pitch), ops.Heads(x, off + hq * d, pitch), be.upload_array(wq), None if d == 96 else
                  be.upload_array(wk), rope, be.upload_array(pos) if rot else None, ops.Heads(q_out), ops.Heads(k_out, 3))
    raw = be.download_array(k_out, np.uint8)
    assert (raw[:3 * es] == 0xAB).all()
    for got, heads, w in ((be.download_array(q_out, np.uint8), slice(0, hq), wq), (raw[3 * es:], slice(hq, None), None if d == 96 else wk)):
        w64 = None if w is None else w.astype(np.float64)
        want = K.turn(K.norm(rows[:, heads], kind, w64, 1e-5), pos, freqs(rot), rot, nb)
        tol = rope_tolerance(rows[:, heads], kind, w64, 1e-5, want, rot, nb, dtype)
        diff = np.abs(values(got, dtype).reshape(want.shape) - want)
        assert (diff <= tol).all(), (diff / tol).max()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("d,rot", [(64, 64), (128, 128), (128, 64)])
def test_without_a_norm_nothing_weighs(be, dtype, d, rot):
    """Weights that a call without a norm gets change nothing, in any of its outputs."""
    t = Setup(be, d + rot, 2, 60, 2, 16, d)
    hq, n = 4, [40, 20]
    x, xv = put(be, t.rng.normal(0, 1, (sum(n), hq + 4, d)), dtype)
    rows, pos = xv.reshape(sum(n), hq + 4, d), np.r_[np.arange(40), np.arange(20)].astype(np.int32)
    w, rope = be.upload_array(np.full(d, 3, np.float32)), ops.prepare_rope(be, freqs(rot))
    want = K.turn(rows[:, :hq], pos, freqs(rot), rot, False)
    tol = rope_tolerance(rows[:, :hq], 0, None, 1e-5, want, rot, False, dtype)
    desc = ops.HeadDesc(hq, 2, d, rot, R.DTYPES[dtype], 0)
    out = be.alloc(want.size * (4 if dtype == "f32" else 2))

    def close():
        assert (np.abs(values(be.download_array(out, np.uint8), dtype).reshape(want.shape) - want) <= tol).all()
    at = lambda h: ops.Heads(x, h * d, (hq + 4) * d)
    ops.norm_rope(be, desc, sum(n), at(0), None, w, w, rope, be.upload_array(pos), ops.Heads(out), None)
    close()
    t.lens[:] = n
    seqs, caches = t.sequences(n), []
    for weight in (None, w):
        ops.append_kv(be, desc, t.cache, seqs, at(hq), at(hq + 2), weight, rope, at(0), weight, ops.Heads(out))
        close()
        caches.append(np.concatenate([be.download_array(b, np.uint8) for b in (t.k, t.v, t.s)]))
    np.testing.assert_array_equal(*caches)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_norm_rope_in_place_and_alone(be, dtype):
    n, hq, d = 37, 5, 128
    rng = np.random.default_rng(3)
    x, xv = put(be, rng.normal(0, 1, n * hq * d), dtype)
    y = be.alloc(x.len_bytes())
    pos = be.upload_array(np.arange(n, dtype=np.int32))
    rope = ops.prepare_rope(be, freqs(d))
    desc = ops.HeadDesc(hq, hq, d, d, R.DTYPES[dtype], ops.NORM_RMS)
    ops.norm_rope(be, desc, n, ops.Heads(x), None, None, None, rope, pos, ops.Heads(y), None)
    a = be.download_array(y, np.uint8)
    ops.norm_rope(be, desc, n, None, ops.Heads(x), None, None, rope, pos, None, ops.Heads(y))
    np.testing.assert_array_equal(be.download_array(y, np.uint8), a)
    ops.norm_rope(be, desc, n, ops.Heads(x), None, None, None, rope, pos, ops.Heads(x), None)
    np.testing.assert_array_equal(be.download_array(x, np.uint8), a)


# ---- append and read

class Setup:
    """A cache on the device and its float64 twin; sequences with pages of their own, in any order."""

    def __init__(self, be, seed, seqs, longest, hk, page, d):
        self.be, self.rng = be, np.random.default_rng(seed)
        self.width = -(-longest // page) + 1
        pages = seqs * self.width + 2
        self.ref = K.Cache(self.rng, pages, hk, page, d)
        self.k, self.v, self.s = (be.upload_array(a) for a in (self.ref.k, self.ref.v, self.ref.s))
        self.cache = ops.KvCache(self.k, self.v, self.s, pages, hk, page, d)
        self.pages = self.rng.permutation(pages)[:seqs * self.width].reshape(seqs, self.width).astype(np.int32)
        self.lens = np.zeros(seqs, np.int32)
        self.hk, self.d, self.page, self.seqs = hk, d, page, seqs

    def sequences(self, n, extra=0, uniform=False):
        """Of n[s] rows each, `extra` rows behind the last."""
        used = -(-self.lens // self.page)
        table = np.where(np.arange(self.width) < used[:, None], self.pages, -7).astype(np.int32)  # the others are not looked at
        starts = np.concatenate([[0], np.cumsum(n)]).astype(np.int32)
        self.starts = starts
        up = self.be.upload_array
        return ops.Sequences(up(table), up(self.lens), None if uniform else up(starts), self.seqs, int(starts[-1]) + extra, self.width)

    def check(self):
        np.testing.assert_array_equal(self.be.download_array(self.s, np.uint8).reshape(self.ref.s.shape), self.ref.s)
        np.testing.assert_array_equal(self.be.download_array(self.k, np.uint8).reshape(self.ref.k.shape), self.ref.k)
        np.testing.assert_array_equal(self.be.download_array(self.v, np.uint8).reshape(self.ref.v.shape), self.ref.v)


def near(got, want, tol):
    """Within the tolerance; where the definition gives NaN (rows whose f16 overflowed), NaN."""
    np.testing.assert_array_equal(np.isnan(got), np.isnan(want))
    ok = np.isnan(want) | (np.abs(got - want) <= tol)
    assert ok.all(), (np.abs(got - want) / tol)[~np.isnan(want)].max()


def append(t, desc, dtype, n, spoil=None, extra=0, uniform=False, gap=0, with_q=True, sizes=1.0):
    """One append_kv of n[s] rows of each sequence on both sides; returns (queries out, queries wanted, tolerance)."""
    be, rng, hq, hk, d = t.be, t.rng, desc.q_heads, t.hk, t.d
    n = np.asarray(n)
    t.lens = (t.lens + n).astype(np.int32)
    seqs = t.sequences(n, extra, uniform)
    rows = int(n.sum()) + extra
    pitch = (hq + 2 * hk) * d + gap
    x = rng.normal(0, 1, (rows, pitch)) * np.exp(rng.normal(0, 1, pitch)) * sizes
    if spoil:
        spoil(x.reshape(-1)[:rows * pitch].reshape(rows, pitch)[:, :(hq + 2 * hk) * d].reshape(rows, -1, d))
    buf, xv = put(be, x, dtype)
    xv = xv.reshape(rows, pitch)[:, :(hq + 2 * hk) * d].reshape(rows, -1, d)
    wq, wk = rng.normal(1, 0.3, (2, d)).astype(np.float32)
    es = 4 if dtype == "f32" else 2
    q_out = be.upload_array(np.full(rows * hq * d * es, 0xAB, np.uint8))
    rope = ops.prepare_rope(be, freqs(desc.rot_dim)) if desc.rot_dim else None
    ops.append_kv(be, desc, t.cache, seqs, ops.Heads(buf, hq * d, pitch), ops.Heads(buf, (hq + hk) * d, pitch), be.upload_array(wk), rope,
                  ops.Heads(buf, 0, pitch) if with_q else None, be.upload_array(wq) if with_q else None, ops.Heads(q_out) if with_q else None)
    total = int(n.sum())
    pos = np.concatenate([np.arange(t.lens[s] - n[s], t.lens[s]) for s in range(t.seqs)])
    f, nb = freqs(desc.rot_dim), bool(desc.neighbours)
    with np.errstate(invalid="ignore"):
        k = K.turn(K.norm(xv[:total, hq:hq + hk], desc.norm, wk.astype(np.float64), 1e-5), pos, f, desc.rot_dim, nb)
        v = xv[:total, hq + hk:]
        for s in range(t.seqs):
            a, b = t.starts[s], t.starts[s + 1]
            t.ref.append(t.pages[s], int(t.lens[s] - n[s]), k[a:b], v[a:b])
        q = xv[:total, :hq]
        want = K.turn(K.norm(q, desc.norm, wq.astype(np.float64), 1e-5), pos, f, desc.rot_dim, nb)
    raw = be.download_array(q_out, np.uint8)
    assert (raw[total * hq * d * es if with_q else 0:] == 0xAB).all()  # rows of no sequence
    return values(raw[:total * hq * d * es], dtype).reshape(want.shape), want, \
        rope_tolerance(q, desc.norm, wq.astype(np.float64), 1e-5, want, desc.rot_dim, nb, dtype)


APPENDS = [  # seqs, hq, hk, page, d, rot, neighbours, norm, rows of each call
    (1, 4, 1, 16, 128, 128, False, 1, [[1]] * 20),
    (3, 2, 2, 32, 64, 64, True, 1, [[5, 0, 33], [1, 1, 1], [0, 31, 64], [2, 1, 0]]),
    (2, 5, 1, 64, 128, 64, False, 2, [[0, 130], [1, 62], [63, 64], [1, 1]]),
    (5, 8, 8, 128, 64, 32, True, 0, [[128, 1, 127, 129, 300], [1, 127, 1, 1, 1]]),
    (40, 2, 1, 16, 128, 128, False, 1, [[i % 4 for i in range(40)], [17] * 40]),
    (2, 3, 3, 16, 128, 0, False, 0, [[7, 16], [10, 1]])]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("case", range(len(APPENDS)))
def test_append(be, dtype, case):
    seqs, hq, hk, page, d, rot, nb, kind, calls = APPENDS[case]
    t = Setup(be, case, seqs, max(sum(c[s] for c in calls) for s in range(seqs)), hk, page, d)
    desc = ops.HeadDesc(hq, hk, d, rot, R.DTYPES[dtype], kind, 1e-5, nb)
    for i, n in enumerate(calls):
        # sizes that grow by call: blocks take larger scales, their codes are rounded again
        got, want, tol = append(t, desc, dtype, n, extra=case % 3, gap=[0, 8, 3][case % 3], uniform=False, with_q=i != 1,
                                sizes=2.0 ** (3 * i if i % 2 else -i))
        t.check()
        if i != 1:
            near(got, want, tol)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_append_the_same_number_to_each(be, dtype):
    t = Setup(be, 9, 6, 100, 2, 32, 128)
    desc = ops.HeadDesc(4, 2, 128, 128, R.DTYPES[dtype], ops.NORM_RMS)
    append(t, desc, dtype, [9, 31, 32, 33, 50, 0])
    for n in (1, 1, 3):
        got, want, tol = append(t, desc, dtype, [n] * 6, uniform=True)
        t.check()
        near(got, want, tol)


@pytest.mark.parametrize("kind", [0, 1])
def test_append_of_what_is_no_number(be, kind):
    """A NaN or an infinity in a token's key or value: that head's token alone."""
    t = Setup(be, 4, 2, 80, 3, 16, 64)
    hq = 3
    desc = ops.HeadDesc(hq, 3, 64, 64, ops.F32, kind)
    append(t, desc, "f32", [10, 40])

    def spoil(x):  # [rows, heads, d]
        x[0, hq, 5], x[1, hq + 1, 0], x[2, hq + 4, 63], x[3, hq + 5, 9], x[25, hq, 1] = np.nan, np.inf, np.nan, -np.inf, -np.inf

    append(t, desc, "f32", [23, 9], spoil=spoil, with_q=False)
    t.check()
    bad = (t.ref.k == 0x7F).all(-1)
    assert bad.sum() >= 5


def test_append_extremes(be):
    """Sizes at the ends of the scales' range and beyond, zeros, values at the borders of codes and of scales."""
    t = Setup(be, 5, 1, 400, 1, 32, 64)
    desc = ops.HeadDesc(1, 1, 64, 0, ops.F32, 0)
    edge = np.concatenate([K.MID, K.MAGS, -K.MID])[:64 * 5].astype(np.float64)

    def fill(v):
        def spoil(x):
            x[:] = v(x)
        return spoil

    for v in (lambda x: x * 0, lambda x: x * 1e-30, lambda x: np.resize(edge, x.shape), lambda x: np.resize(edge * 2.0 ** 63, x.shape),
              lambda x: x * 1e30, lambda x: np.full(x.shape, 448.0), lambda x: np.full(x.shape, 448.0) * (1 + 2.0 ** -23),
              lambda x: np.resize(edge * 2.0 ** -66, x.shape), lambda x: np.full(x.shape, 3.0e38)):
        append(t, desc, "f32", [33], spoil=fill(v), with_q=False)
        t.check()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("page,d,hk", [(16, 64, 3), (64, 128, 1), (128, 128, 2)])
def test_read(be, dtype, page, d, hk):
    t = Setup(be, 6, 4, 300, hk, page, d)
    desc = ops.HeadDesc(hk, hk, d, d, ops.F32, ops.NORM_RMS)
    append(t, desc, "f32", [300, 1, 0, 77], with_q=False, sizes=0.01)
    n = np.array([300, 1, 2, 30])  # two rows of an empty sequence: no tokens
    seqs = t.sequences(n, extra=2)
    es, rows = (4 if dtype == "f32" else 2), int(n.sum()) + 2
    pitch = hk * d + 5
    out = [be.upload_array(np.full(((rows - 1) * pitch + hk * d + 1) * es, 0xAB, np.uint8)) for _ in range(2)]
    ops.read_kv(be, t.cache, seqs, R.DTYPES[dtype], ops.Heads(out[0], 1, pitch), ops.Heads(out[1], 1, pitch))
    for which in range(2):
        raw = be.download_array(out[which], np.uint8)
        got = values(raw[es:], dtype)
        got = np.pad(got, (0, rows * pitch - got.size)).reshape(rows, pitch)
        sentinel = values(np.full(es, 0xAB, np.uint8), dtype)[0]
        assert (got[:-1, hk * d:] == sentinel).all() and (got[-2:, :hk * d] == sentinel).all()
        for s in range(4):
            length = int(t.lens[s])
            want = t.ref.read(which, t.pages[s], length)[max(0, length - n[s]):]
            want = R.to_type(np.concatenate([np.zeros((n[s] - len(want), hk, d)), want]).reshape(-1), dtype)[1]
            np.testing.assert_array_equal(got[t.starts[s]:t.starts[s + 1], :hk * d].reshape(-1), want)
    one = be.upload_array(np.full(out[0].len_bytes(), 0xAB, np.uint8))
    ops.read_kv(be, t.cache, seqs, R.DTYPES[dtype], None, ops.Heads(one, 1, pitch))
    np.testing.assert_array_equal(be.download_array(one, np.uint8), raw)
    ops.read_kv(be, t.cache, seqs, R.DTYPES[dtype], ops.Heads(one, 1, pitch), None)


def test_bad_lengths_starts_and_pages_are_reported(be):
    """Not followed (each is brought into bounds by the kernel), and reported once."""
    t = Setup(be, 7, 2, 64, 1, 16, 64)
    desc = ops.HeadDesc(1, 1, 64, 64, ops.F16, ops.NORM_RMS)
    append(t, desc, "f16", [40, 20])
    x = be.upload_array(np.zeros(3 * 2 * 64, np.float16))
    up = be.upload_array
    rope = ops.prepare_rope(be, freqs(64))
    good = dict(table=t.pages, lens=np.array([41, 22], np.int32), starts=np.array([0, 1, 3], np.int32))
    for change in (dict(lens=np.array([41, -3], np.int32)), dict(lens=np.array([1 << 30, 22], np.int32)),
                   dict(starts=np.array([0, -5, 3], np.int32)), dict(starts=np.array([0, 2, 1], np.int32)),
                   dict(starts=np.array([0, 1, 400], np.int32)), dict(table=np.full_like(t.pages, 1 << 20)),
                   dict(table=np.full_like(t.pages, -1))):
        a = {**good, **change}
        seqs = ops.Sequences(up(a["table"]), up(a["lens"]), up(a["starts"]), 2, 3, t.width)
        for call in (lambda: ops.append_kv(be, desc, t.cache, seqs, ops.Heads(x, 0, 128), ops.Heads(x, 64, 128), None, rope),
                     lambda: ops.read_kv(be, t.cache, seqs, ops.F16, ops.Heads(x), None),
                     lambda: ops.attention_kv8(be, ops.AttentionDesc(1, ops.F16, 1.0), t.cache, seqs, ops.Heads(x), ops.Heads(x, 192))):
            call()
            with pytest.raises(dw.BackendError) as e:
                be.synchronize(20000)
            assert e.value.status == dw.ops.L.DW_ERR_DEVICE
            be.synchronize(20000)
    seqs = ops.Sequences(up(t.pages), up(t.lens), None, 2, 2, t.width)
    ops.read_kv(be, t.cache, seqs, ops.F16, ops.Heads(x), None)
    be.synchronize(20000)


def test_refusals(be):
    t = Setup(be, 8, 2, 64, 2, 16, 64)
    append(t, ops.HeadDesc(4, 2, 64, 64, ops.F16, ops.NORM_RMS), "f16", [40, 20])
    L = ops.L
    up, rope = be.upload_array, ops.prepare_rope(be, freqs(64))
    x = up(np.zeros(2 * 8 * 64, np.float16))
    pos, w = up(np.zeros(2, np.int32)), up(np.ones(64, np.float32))
    seqs = t.sequences([1, 1])
    H = ops.Heads

    def refused(status, call):
        before = be.launch_count()
        with pytest.raises(dw.BackendError) as e:
            call()
        assert e.value.status == status and e.value.message and be.launch_count() == before

    def rope_call(desc=(4, 2, 64, 64, ops.F16, 1), tokens=2, q=H(x, 0, 512), k=H(x, 256, 512), wq=w, r=rope, p=pos, qo=H(x, 0, 512),
                  ko=H(x, 256, 512), **kw):
        return lambda: ops.norm_rope(be, ops.HeadDesc(*desc, **kw), tokens, q, k, wq, None, r, p, qo, ko)

    bad, size, un = L.DW_ERR_INVALID_ARG, L.DW_ERR_SIZE_MISMATCH, L.DW_ERR_UNSUPPORTED
    for status, call in (
            (bad, rope_call(desc=(0, 2, 64, 64, ops.F16, 1))), (un, rope_call(desc=(4, 2, 63, 62, ops.F16, 1))),
            (un, rope_call(desc=(4, 2, 514, 64, ops.F16, 1))), (bad, rope_call(desc=(4, 2, 64, 66, ops.F16, 1))),
            (bad, rope_call(desc=(4, 2, 64, 63, ops.F16, 1))), (bad, rope_call(desc=(4, 2, 64, 64, 3, 1))),
            (bad, rope_call(desc=(4, 2, 64, 64, ops.F16, 3))), (bad, rope_call(eps=-1.0)), (bad, rope_call(eps=float("nan"))),
            (bad, rope_call(tokens=0)), (bad, rope_call(tokens=1 << 31)), (size, rope_call(tokens=3)), (bad, rope_call(q=H(x, 0, 200))),
            (size, rope_call(q=H(x, 257, 512))), (bad, rope_call(q=None)), (bad, rope_call(qo=None)),
            (bad, rope_call(q=None, k=None, qo=None, ko=None)), (bad, rope_call(r=None)), (bad, rope_call(p=None)),
            (size, rope_call(r=up(np.zeros(33, np.uint64)))), (size, rope_call(p=up(np.zeros(3, np.int32)))),
            (size, rope_call(wq=up(np.ones(63, np.float32)))), (bad, rope_call(desc=(4, 2, 64, 0, ops.F16, 1))),
            (bad, rope_call(q=H(None))), (size, rope_call(q=H(x, 1 << 59)))):
        refused(status, call)
    rope_call()()

    cache = lambda **kw: ops.KvCache(**{**dict(k=t.k, v=t.v, scales=t.s, pages=t.ref.k.shape[0], kv_heads=2, page_tokens=16, head_dim=64), **kw})
    sq = lambda **kw: ops.Sequences(**{**dict(table=seqs.keep[0], lens=seqs.keep[1], starts=seqs.keep[2], seqs=2, tokens=2, width=t.width), **kw})

    def app(desc=(4, 2, 64, 64, ops.F16, 1), c=t.cache, s=seqs, k=H(x, 0, 512), v=H(x, 128, 512), r=rope, q=None, qo=None):
        return lambda: ops.append_kv(be, ops.HeadDesc(*desc), c, s, k, v, w, r, q, None, qo)

    def att(desc=(4, ops.F16, 1.0), c=t.cache, s=seqs, q=H(x), o=H(x)):
        return lambda: ops.attention_kv8(be, ops.AttentionDesc(*desc), c, s, q, o)

    def read(c=t.cache, s=seqs, dtype=ops.F16, k=H(x), v=None):
        return lambda: ops.read_kv(be, c, s, dtype, k, v)

    caches = [(bad, dict(k=None)), (bad, dict(scales=None)), (bad, dict(pages=0)), (bad, dict(kv_heads=0)), (un, dict(page_tokens=8)),
              (un, dict(page_tokens=48)), (un, dict(head_dim=96)), (size, dict(pages=t.ref.k.shape[0] + 1)), (size, dict(v=t.s)),
              (un, dict(pages=1 << 30))]
    sequences = [(bad, dict(seqs=0)), (bad, dict(tokens=0)), (bad, dict(width=0)), (bad, dict(table=None)), (bad, dict(lens=None)),
                 (size, dict(width=t.width + 1)), (size, dict(seqs=3)), (bad, dict(starts=None, tokens=3)), (size, dict(starts=seqs.keep[1])),
                 (un, dict(width=1 << 28))]
    for make in (lambda **k: app(**k), lambda **k: att(**k), lambda **k: read(**k)):
        for status, kw in caches:
            refused(status, make(c=cache(**kw)))
        for status, kw in sequences:
            refused(status, make(s=sq(**kw)))
    for status, call in (
            (bad, app(desc=(4, 1, 64, 64, ops.F16, 1))), (bad, app(k=None)), (bad, app(v=H(None))), (size, app(v=H(x, 400, 600))),
            (bad, app(q=H(x))), (bad, app(qo=H(x))), (bad, app(desc=(4, 2, 128, 128, ops.F16, 1), r=ops.prepare_rope(be, freqs(128)))),
            (un, att(desc=(4, ops.F32, 1.0))), (bad, att(desc=(3, ops.F16, 1.0))), (bad, att(desc=(0, ops.F16, 1.0))),
            (bad, att(desc=(4, ops.F16, -1.0))), (bad, att(desc=(4, ops.F16, float("nan")))), (bad, att(desc=(4, ops.F16, float("inf")))),
            (bad, att(desc=(4, ops.F16, 1.0, True, -1))), (bad, att(desc=(4, ops.F16, 1.0, False, 5))), (bad, att(q=H(None))),
            (size, att(q=H(x, 513))), (bad, att(o=H(x, 0, 255))), (bad, read(k=None)), (bad, read(dtype=7)), (size, read(k=H(x, 900)))):
        refused(status, call)
    t128 = Setup(be, 8, 1, 64, 1, 16, 128)
    t128.lens[:] = 1
    refused(un, lambda: ops.append_kv(be, ops.HeadDesc(1, 1, 128, 62, ops.F16), t128.cache, t128.sequences([1]), H(x), H(x), None,
                                      ops.prepare_rope(be, freqs(62))))
    for f in ([float("nan")], [float("inf")], [], [1.0] * 257):
        refused(bad, lambda: ops.prepare_rope(be, f))
    app()(), att()(), read()()
    be.synchronize(20000)
