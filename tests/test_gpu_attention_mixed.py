"""Calls whose sequences have very different numbers of rows: a prompt beside single tokens, on either kernel; captured
with starts of its own and replayed with others."""
import ctypes

import numpy as np
import pytest

import dragonwing_edge_rs_b200 as dw
from dragonwing_edge_rs_b200 import ops
from tests.test_gpu_attention import attend, check, filled
from tests.test_gpu_kv_heads import values

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def be():
    with dw.CudaBackend(0) as b:
        yield b


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("n,group", [([260] + [1] * 12, 4), ([1] * 40 + [150, 0], 2), ([1, 90, 1, 1, 0, 1], 5), ([2, 1, 400], 1)])
@pytest.mark.parametrize("window", [0, 37])
def test_a_prompt_beside_single_tokens(be, dtype, n, group, window):
    lens = [m + 13 * (i % 7) for i, m in enumerate(n)]
    t = filled(be, len(n), lens, 2, 16, 64)
    attend(t, 2 * group, dtype, n, window=window, extra=2)


@pytest.mark.parametrize("rows", [9, 200])
def test_captured_and_replayed_with_other_starts(be, rows):
    """Ragged rows: the graph's call gives the eager call's bits for other starts and lengths, rows of no sequence in
    front and behind among them."""
    t = filled(be, rows, [400, 300, 250, 90], 1, 32, 128)
    lib, up = ops.L.load(), be.upload_array
    q = up(t.rng.normal(0, 1, rows * 4 * 128).astype(np.float16))
    lens, starts = up(t.lens), up(np.zeros(5, np.int32))
    seqs = ops.Sequences(up(t.pages), lens, starts, 4, rows, t.width)
    desc = ops.AttentionDesc(4, ops.F16, 128 ** -0.5)
    a, b = (be.alloc(q.len_bytes()) for _ in range(2))
    g = ctypes.c_void_p()
    be._check(lib.dw_capture_begin(be.handle))
    ops.attention_kv8(be, desc, t.cache, seqs, ops.Heads(q), ops.Heads(a))
    be._check(lib.dw_capture_end(be.handle, ctypes.byref(g)))
    qv = values(be.download_array(q, np.uint8), "f16").reshape(rows, 4, 128)
    for cut, length in (([0, 1, 2, 3, rows], [400, 300, 250, 90]), ([0, rows, rows, rows, rows], [400, 0, 0, 0]),
                        ([2, 2, rows - 3, rows - 1, rows - 1], [7, 250, 3, 90]), ([0, 0, 0, 0, 0], [400, 300, 250, 90])):
        for buf in (a, b):
            be.upload(buf, np.full(q.len_bytes(), 0x3C, np.uint8))
        be.upload(lens, np.asarray(length, np.int32))
        be.upload(starts, np.asarray(cut, np.int32))
        be._check(lib.dw_graph_launch(be.handle, g))
        ops.attention_kv8(be, desc, t.cache, seqs, ops.Heads(q), ops.Heads(b))
        be.synchronize(20000)
        raw = be.download_array(b, np.uint8)
        np.testing.assert_array_equal(be.download_array(a, np.uint8), raw)
        t.lens, t.starts = np.asarray(length, np.int32), np.asarray(cut)
        got = values(raw, "f16").reshape(rows, 4, 128)
        check(t, desc, "f16", None, qv, got)
        for out in (raw.reshape(rows, -1)[:cut[0]], raw.reshape(rows, -1)[cut[4]:]):
            assert (out == 0x3C).all()
    lib.dw_graph_destroy(g)
