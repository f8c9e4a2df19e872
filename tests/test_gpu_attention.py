"""Attention over the paged 8-bit cache against float64 on the same cached values, and the run of appends and
attention that a served layer makes."""
import ctypes

import numpy as np
import pytest

import dragonwing_edge_rs_b200 as dw
from dragonwing_edge_rs_b200 import ops
from tests import _kv_ref as K
from tests import _mxfp4_ref as R
from tests.test_gpu_kv_heads import HALF_STEP, Setup, append, put, values

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def be():
    with dw.CudaBackend(0) as b:
        yield b


def tolerance(want, mean, big, mass, length, d, dtype):
    """A logit: d exact products summed in f32 with at most a whole last place lost in each of d / 8 sums, of their
    absolute sum; its scaling, the value scale's addition and the maximum's: four roundings of |t| + 64 + 14 in units
    of log2; 2^x 2^-22.  A weight is off by that, twice (numerator and denominator), and by its cut to 11 bits: both sums
    take the cut weights w (1 - e), 0 <= e < 2^-10, and sum w (v - out) = 0, so sum w (e - 2^-11) (v - out) / sum w, at
    most 2^-11 (mean + |out|), is what that does.
    The values' sum: at most a whole last place in each of length / 8 + 32 sums and joins.  Then the result's rounding."""
    weight = 2.0 ** -11 + 2 * (d / 8 * 2.0 ** -23 * mass + 4 * 2.0 ** -23 * (2 * big + 78) + 2.0 ** -22)
    tol = (weight * 1.1 + (length / 8 + 32) * 2.0 ** -23) * mean + 2.0 ** -11 * np.abs(want)
    floor = {"f16": 2.0 ** -25, "bf16": 1e-40}[dtype]
    return tol + HALF_STEP[dtype] * (np.abs(want) + tol) + floor + length * 2.0 ** -38 * np.nan_to_num(mean).max(initial=0.0)


def check(t, desc, dtype, n, q, got, first=0):
    """Rows of each sequence against float64."""
    for s in range(t.seqs):
        a, b, length = t.starts[s], t.starts[s + 1], int(t.lens[s])
        k, v = t.ref.read(0, t.pages[s], length), t.ref.read(1, t.pages[s], length)
        with np.errstate(invalid="ignore"):
            want, *how = K.attention(q[a:b], k, v, length, float(np.float32(desc.scale)), desc.causal, desc.window)
        assert np.array_equal(np.isnan(got[a:b]), np.isnan(want)), s
        tol = tolerance(want, *how, length, t.d, dtype)
        ok = np.isnan(want) | (np.abs(got[a:b] - want) <= tol)
        assert ok.all(), (s, (np.abs(got[a:b] - want) / tol)[~np.isnan(want)].max())


def attend(t, hq, dtype, n, causal=True, window=0, scale=None, extra=0, uniform=False, gap=0, offset=0, in_place=False, q=None):
    be, rng, d = t.be, t.rng, t.d
    n = np.asarray(n)
    seqs = t.sequences(n, extra, uniform)
    rows = int(n.sum()) + extra
    pitch = hq * d + gap
    x = rng.normal(0, 1.5, rows * pitch + offset) if q is None else q
    buf, xv = put(be, x, dtype)
    xv = xv[offset:].reshape(rows, pitch)[:, :hq * d].reshape(rows, hq, d)
    out = buf if in_place else be.upload_array(np.full((rows * pitch + offset) * 2, 0xAB, np.uint8))
    desc = ops.AttentionDesc(hq, R.DTYPES[dtype], 1 / np.sqrt(d) if scale is None else scale, causal, window)
    ops.attention_kv8(be, desc, t.cache, seqs, ops.Heads(buf, offset, pitch), ops.Heads(out, offset, pitch))
    raw = be.download_array(out, np.uint8)
    got = values(raw[2 * offset:], dtype).reshape(rows, pitch)
    if not in_place:
        assert (raw[:2 * offset] == 0xAB).all()
        sentinel = values(np.full(2, 0xAB, np.uint8), dtype)[0]
        assert (got[:, hq * d:] == sentinel).all() and (got[int(n.sum()):] == sentinel).all()
    got = got[:, :hq * d].reshape(rows, hq, d)
    check(t, desc, dtype, n, xv, got)
    return raw


def filled(be, seed, lens, hk, page, d, spoil=None):
    """Sequences of the given lengths; pages behind them hold anything."""
    t = Setup(be, seed, len(lens), max(max(lens), 1), hk, page, d)
    append(t, ops.HeadDesc(hk, hk, d, 0, ops.F32, 0), "f32", lens, with_q=False, spoil=spoil)
    return t


LENS = [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 129, 300, 1000, 0]


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("page,d,hk,group", [(16, 128, 1, 4), (32, 64, 2, 1), (64, 128, 2, 8), (128, 64, 1, 5), (16, 64, 1, 16), (64, 128, 1, 33)])
def test_single_tokens(be, dtype, page, d, hk, group):
    t = filled(be, page + d, LENS, hk, page, d)
    attend(t, hk * group, dtype, [1] * len(LENS), uniform=True)
    attend(t, hk * group, dtype, [1] * len(LENS), window=20, extra=3, gap=8)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("lens", [[1], [5000], [20000], [700, 3000]])
def test_few_long_sequences(be, dtype, lens):
    """The CTAs of a cluster share a sequence."""
    t = filled(be, len(lens), lens, 1, 32, 128)
    attend(t, 4, dtype, [1] * len(lens), uniform=True)
    attend(t, 3, dtype, [1] * len(lens), window=999)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("n", [[5] * 4, [1, 7, 0, 3], [40, 1, 200, 17], [33, 0, 0, 0]])
@pytest.mark.parametrize("causal,window", [(True, 0), (False, 0), (True, 10), (True, 1)])
def test_rows_behind_a_cache(be, dtype, n, causal, window):
    t = filled(be, sum(n), [x + o for x, o in zip(n, (0, 31, 5, 100))], 2, 16, 64)
    attend(t, 6, dtype, n, causal, window, extra=2, gap=3, offset=1)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("page,d,hk,group", [(16, 64, 1, 1), (64, 128, 1, 4), (32, 128, 2, 7), (128, 64, 2, 8), (64, 128, 1, 1)])
@pytest.mark.parametrize("lens,n", [([600], [600]), ([333, 40, 900], [333, 40, 200]), ([1, 129, 257], [1, 129, 256])])
def test_prompts(be, dtype, page, d, hk, group, lens, n):
    t = filled(be, page + d + len(n), lens, hk, page, d)
    attend(t, hk * group, dtype, n)
    if group < 7:
        attend(t, hk * group, dtype, n, window=100, extra=1)
        attend(t, hk * group, dtype, n, causal=False, gap=16)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("page,d,hk,group,lens,n", [(64, 128, 1, 4, [4000], [70]), (16, 64, 2, 5, [1500], [60]), (32, 128, 1, 3, [2100, 900, 65], [20, 100, 61]),
                                                    (128, 64, 1, 1, [3000, 40], [257, 3]), (64, 128, 1, 1, [600], [49])])
def test_pieces_of_prompts_behind_long_caches(be, dtype, page, d, hk, group, lens, n):
    """Few blocks of many rows: the CTAs of a cluster share a block's tokens, some with tiles of one half of the rows
    alone or with none."""
    t = filled(be, page + d + len(n), lens, hk, page, d)
    attend(t, hk * group, dtype, n, in_place=True)
    attend(t, hk * group, dtype, n, uniform=len(n) == 1, gap=5, offset=3, in_place=True)
    attend(t, hk * group, dtype, n, window=300, extra=2)
    attend(t, hk * group, dtype, n, causal=False, gap=8)


def test_more_rows_than_tokens(be):
    """Rows before the first position see nothing."""
    t = filled(be, 1, [3, 0, 70], 1, 16, 64)
    raw = attend(t, 2, "f16", [10, 4, 90])
    assert not raw[:7 * 2 * 64 * 2].any()
    t = filled(be, 1, [3, 0, 70], 1, 16, 128)
    attend(t, 2, "bf16", [300, 400, 500])


@pytest.mark.parametrize("n", [3, 300])
def test_in_place_and_again(be, n):
    t = filled(be, 2, [1000, 2000], 2, 64, 128)
    q = t.rng.normal(0, 1, 2 * n * 4 * 128)
    a = attend(t, 4, "bf16", [n, n], q=q)
    b = attend(t, 4, "bf16", [n, n], q=q, in_place=True)
    np.testing.assert_array_equal(a, b)


@pytest.mark.parametrize("n", [1, 4, 150])
@pytest.mark.parametrize("d", [64, 128])
def test_what_is_no_number_stays_with_who_sees_it(be, n, d):
    """Tokens with NaN or infinity in key or value: NaN for the rows and heads that see them, nobody else."""
    def spoil(x):  # rows of three sequences: q, k, v heads of two
        x[0, 2, 3] = np.nan                 # the first token of sequence 0, key of head 0
        x[180, 5, 0] = np.inf               # a late token of sequence 0, value of head 1
        x[200 + 199, 3, 1] = -np.inf        # the last token of sequence 1, key of head 1
    t = filled(be, 3, [200, 200, 200], 2, 16, d, spoil)
    attend(t, 4, "f16", [n] * 3)
    attend(t, 4, "bf16", [n] * 3, window=12)
    attend(t, 4, "f16", [n] * 3, causal=False)
    q = t.rng.normal(0, 1, (3 * n, 4, d))
    q[0, 1, 5], q[-1, 2, 0] = np.nan, np.inf
    attend(t, 4, "f16", [n] * 3, q=q.reshape(-1))
    attend(t, 4, "bf16", [n] * 3, q=q.reshape(-1))


@pytest.mark.parametrize("n", [1, 200])
@pytest.mark.parametrize("size", [2.0 ** -60, 2.0 ** -20, 2.0 ** 20, 2.0 ** 55])
def test_blocks_of_very_different_size(be, n, size):
    """Every second page's values are `size` times the others', the keys' sizes differ too."""
    def spoil(x):
        x[:, 2] *= np.where(np.arange(len(x)) // 16 % 2, 1.0, size)[:, None]
        x[:, 1] *= np.where(np.arange(len(x)) // 16 % 3, 1.0, 2.0 ** -30)[:, None]
    t = filled(be, 4, [700], 1, 16, 64, spoil)
    attend(t, 2, "bf16", [n])


@pytest.mark.parametrize("n", [1, 130])
@pytest.mark.parametrize("dtype,size", [("f16", 2.0 ** -24), ("f16", 6e4), ("bf16", 1e-38), ("bf16", 1e30)])
def test_queries_of_any_size(be, n, dtype, size):
    t = filled(be, 5, [400], 1, 32, 128)
    q = (t.rng.uniform(0.5, 1, n * 2 * 128) * t.rng.choice([-1, 1], n * 2 * 128)) * size
    attend(t, 2, dtype, [n], scale=0.05 / size, q=q)
    attend(t, 2, dtype, [n], scale=0.0, q=q)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_a_layer_step_by_step_and_captured(be, dtype):
    """A prompt, then single tokens, as a served layer runs them: each step against float64; the step captured once
    and replayed with other rows and lengths gives the eager step's bits."""
    hq, hk, d, page = 8, 2, 128, 16
    t = Setup(be, 11, 3, 150, hk, page, d)
    desc = ops.HeadDesc(hq, hk, d, d, R.DTYPES[dtype], ops.NORM_RMS)
    att = ops.AttentionDesc(hq, R.DTYPES[dtype], 1 / np.sqrt(d))
    q, _, _ = append(t, desc, dtype, [100, 3, 31])
    attend(t, hq, dtype, [100, 3, 31], q=q.reshape(-1))
    lib = ops.L.load()
    rng = np.random.default_rng(0)
    up = be.upload_array
    freq = 10000.0 ** (-2.0 * np.arange(d // 2) / d)
    rope, w = ops.prepare_rope(be, freq), up(np.ones(d, np.float32))
    pitch = (hq + 2 * hk) * d
    x, qb, o = be.alloc(3 * pitch * 2), be.alloc(3 * hq * d * 2), be.alloc(3 * hq * d * 2)
    lens, table = up(t.lens), up(t.pages)
    seqs = ops.Sequences(table, lens, None, 3, 3, t.width)

    def step():
        ops.append_kv(be, desc, t.cache, seqs, ops.Heads(x, hq * d, pitch), ops.Heads(x, (hq + hk) * d, pitch), w, rope,
                      ops.Heads(x, 0, pitch), w, ops.Heads(qb))
        ops.attention_kv8(be, att, t.cache, seqs, ops.Heads(qb), ops.Heads(o))

    g = ctypes.c_void_p()
    be._check(lib.dw_capture_begin(be.handle))
    step()
    be._check(lib.dw_capture_end(be.handle, ctypes.byref(g)))
    for i in range(20):
        t.lens = t.lens + 1
        be.upload(lens, t.lens.astype(np.int32))
        raw, xv = R.to_type(rng.normal(0, 1 + i, 3 * pitch), dtype)
        be.upload(x, raw)
        before = [be.download_array(b, np.uint8) for b in (t.k, t.v, t.s)]
        step()
        eager = [be.download_array(b, np.uint8) for b in (o, t.k, t.v, t.s)]
        for b, was in zip((t.k, t.v, t.s), before):
            be.upload(b, was)
        be._check(lib.dw_graph_launch(be.handle, g))
        for b, want in zip((o, t.k, t.v, t.s), eager):
            np.testing.assert_array_equal(be.download_array(b, np.uint8), want)
        rows = np.asarray(xv, np.float64).reshape(3, -1, d)
        pos = t.lens - 1
        kk = K.turn(K.norm(rows[:, hq:hq + hk], 1, None, 1e-5), pos, freq, d, False)
        for s in range(3):
            t.ref.append(t.pages[s], int(pos[s]), kk[s:s + 1], rows[s:s + 1, hq + hk:])
        t.check()
        t.starts = np.arange(4)
        check(t, att, dtype, [1] * 3, values(be.download_array(qb, np.uint8), dtype).reshape(3, hq, d),
              values(eager[0], dtype).reshape(3, hq, d))
    lib.dw_graph_destroy(g)


def test_shared_pages_and_two_backends(be):
    """Sequences that share a prefix's pages; two backends (streams) on one cache at once."""
    t = filled(be, 12, [320, 320], 1, 64, 64)
    t.pages[1, :4] = t.pages[0, :4]
    want = attend(t, 4, "f16", [2, 2], uniform=True, q=np.ones(2 * 2 * 4 * 64))
    with dw.CudaBackend(0) as other:
        q = other.upload_array(np.ones(2 * 2 * 4 * 64, np.float16))
        outs = [be.alloc(q.len_bytes()) for _ in range(20)]
        seqs = t.sequences([2, 2], uniform=True)
        desc = ops.AttentionDesc(4, ops.F16, 1 / 8)
        for i, out in enumerate(outs):
            ops.attention_kv8(be if i % 2 else other, desc, t.cache, seqs, ops.Heads(q), ops.Heads(out))
        be.synchronize(), other.synchronize()
        for out in outs:
            np.testing.assert_array_equal(be.download_array(out, np.uint8), want)


@pytest.mark.parametrize("n", [20, 90])
def test_captured_pieces_of_prompts_beside_another_backend(be, n):
    """Few and many rows whose tokens a cluster shares: a captured call, replayed at other lengths (one of them 0, one
    shorter than its rows), gives the eager call's bits while another backend makes the same calls."""
    t = filled(be, n, [2500, 1700], 1, 32, 128)
    lib, up, bytes_ = ops.L.load(), be.upload_array, 2 * n * 2 * 128 * 2
    q = up(t.rng.normal(0, 1, bytes_ // 2).astype(np.float16))
    lens, table = up(t.lens), up(t.pages)
    seqs = ops.Sequences(table, lens, None, 2, 2 * n, t.width)
    desc = ops.AttentionDesc(2, ops.F16, 128 ** -0.5)
    a, b, c = (be.alloc(bytes_) for _ in range(3))
    g = ctypes.c_void_p()
    be._check(lib.dw_capture_begin(be.handle))
    ops.attention_kv8(be, desc, t.cache, seqs, ops.Heads(q), ops.Heads(a))
    be._check(lib.dw_capture_end(be.handle, ctypes.byref(g)))
    with dw.CudaBackend(0) as other:
        for now in ([2500, 1700], [1, 1700], [0, 64], [n - 1, n], [2499, 3]):
            be.upload(lens, np.asarray(now, np.int32))
            be.synchronize()
            for _ in range(5):
                be._check(lib.dw_graph_launch(be.handle, g))
                ops.attention_kv8(other, desc, t.cache, seqs, ops.Heads(q), ops.Heads(c))
            ops.attention_kv8(be, desc, t.cache, seqs, ops.Heads(q), ops.Heads(b))
            be.synchronize(), other.synchronize()
            want = be.download_array(b, np.uint8)
            np.testing.assert_array_equal(be.download_array(a, np.uint8), want)
            np.testing.assert_array_equal(be.download_array(c, np.uint8), want)
            t.lens[:], t.starts = now, np.array([0, n, 2 * n])
            check(t, desc, "f16", n, values(be.download_array(q, np.uint8), "f16").reshape(2 * n, 2, 128), values(want, "f16").reshape(2 * n, 2, 128))
    lib.dw_graph_destroy(g)
