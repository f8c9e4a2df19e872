"""Appends whose lengths, starts or pages lie outside: reported, and no token of the cache is lost to them."""
import numpy as np
import pytest

import dragonwing_edge_rs_b200 as dw
from dragonwing_edge_rs_b200 import ops
from tests.test_gpu_kv_heads import Setup, append, freqs

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def be():
    with dw.CudaBackend(0) as b:
        yield b


def held(t):
    return [t.be.download_array(b, np.uint8).reshape(r.shape) for b, r in ((t.k, t.ref.k), (t.v, t.ref.v), (t.s, t.ref.s))]


BAD = [  # (what is wrong, of three sequences of 40, 20 and 33 tokens that get 1, 2 and 3; who is appended to all the same)
    (dict(lens=[41, -3, 36]), [0, 2]), (dict(lens=[1 << 30, 22, 36]), [1, 2]), (dict(lens=[41, 22, 16 * 5 + 1]), [0, 1]),
    (dict(starts=[0, -5, 3, 6]), [2]), (dict(starts=[0, 5, 3, 6]), []), (dict(starts=[0, 1, 3, 400]), [0, 1]),
    (dict(starts=[9, 1, 3, 6]), [2]), (dict(pages=[(1, 1, -1)]), [0, 2]), (dict(pages=[(0, 2, 1 << 20), (2, 2, -5)]), [1]),
    (dict(pages=[(0, 2, -1), (1, 1, -1), (2, 2, -1)]), [])]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("case", range(len(BAD)))
def test_nothing_is_written_for_what_lies_outside(be, dtype, case):
    change, good = BAD[case]
    t = Setup(be, case, 3, 64, 2, 16, 64)
    desc = ops.HeadDesc(2, 2, 64, 64, {"f32": ops.F32, "f16": ops.F16, "bf16": ops.BF16}[dtype], ops.NORM_RMS)
    # physical page 0 is a sequence's first
    if 0 not in t.pages[2, :1]:
        swap = t.pages[2, 0]
        t.pages = np.where(t.pages == 0, -2, t.pages)
        t.pages[2, 0] = 0
        t.pages = np.where(t.pages == -2, swap, t.pages).astype(np.int32)
    append(t, desc, dtype, [40, 20, 33], with_q=False)
    t.check()
    before = held(t)
    table = t.pages.copy()
    for s, i, to in change.get("pages", []):
        table[s, i] = to
    n, up = [1, 2, 3], be.upload_array
    seqs = ops.Sequences(up(table), up(np.array(change.get("lens", [41, 22, 36]), np.int32)),
                         up(np.array(change.get("starts", [0, 1, 3, 6]), np.int32)), 3, 6, t.width)
    x = up(np.random.default_rng(1).normal(0, 100, 6 * 4 * 64).astype({"f32": np.float32}.get(dtype, np.float16)))
    ops.append_kv(be, desc, t.cache, seqs, ops.Heads(x, 0, 256), ops.Heads(x, 128, 256), None, ops.prepare_rope(be, freqs(64)))
    with pytest.raises(dw.BackendError) as e:
        be.synchronize(20000)
    assert e.value.status == dw.ops.L.DW_ERR_DEVICE
    be.synchronize(20000)
    after = held(t)
    new = np.zeros(before[0].shape[:1] + (1, 16), bool)  # places that a good sequence's new tokens take, and its blocks
    for s in good:
        old = [40, 20, 33][s]
        for p in range(old, old + n[s]):
            new[t.pages[s, p // 16], 0, p % 16] = True
    blocks = new.any((1, 2))
    for a, b in zip(after, before):
        np.testing.assert_array_equal(a[~blocks], b[~blocks])
    for s in good:  # (values of other sizes than those held: scales grow, and some code of each new token is another)
        page = t.pages[s, [40, 20, 33][s] // 16]
        assert (after[2][page] != before[2][page]).any()


@pytest.mark.parametrize("seqs,rows", [(70, 1), (70, 90), (3, 5)])
@pytest.mark.parametrize("which", ["append", "read", "attend"])
def test_a_descent_anywhere_is_reported(be, seqs, rows, which):
    """One pair of starts out of order, in the middle or at an end, where the sequences around it are empty or not."""
    t = Setup(be, 3, seqs, 120, 1, 16, 64)
    t.lens[:] = 100
    x = be.upload_array(np.zeros(rows * 4 * 64, np.float16))
    up, rng = be.upload_array, np.random.default_rng(rows)
    desc = ops.HeadDesc(1, 1, 64, 0, ops.F16, 0)
    for at in {1, 2, seqs // 2, seqs - 1, seqs}:
        starts = np.sort(rng.integers(0, rows + 1, seqs + 1)).astype(np.int32)
        starts[at - 1], starts[at] = rows, rows - 1
        sq = ops.Sequences(up(t.pages), up(t.lens), up(starts), seqs, rows, t.width)
        if which == "append":
            ops.append_kv(be, desc, t.cache, sq, ops.Heads(x, 0, 128), ops.Heads(x, 64, 128))
        elif which == "read":
            ops.read_kv(be, t.cache, sq, ops.F16, ops.Heads(x), None)
        else:
            ops.attention_kv8(be, ops.AttentionDesc(1, ops.F16, 1.0), t.cache, sq, ops.Heads(x), ops.Heads(x, rows * 64))
        with pytest.raises(dw.BackendError) as e:
            be.synchronize(20000)
        assert e.value.status == dw.ops.L.DW_ERR_DEVICE
    be.synchronize(20000)
