"""Attention in a window over a cache whose pages before the window were given away: their table entries name no page
and their tokens are anybody's."""
import numpy as np
import pytest

import dragonwing_edge_rs_b200 as dw
from dragonwing_edge_rs_b200 import ops
from tests.test_gpu_attention import attend, filled
from tests.test_gpu_kv_heads import append

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def be():
    with dw.CudaBackend(0) as b:
        yield b


def give_away(t, n, window):
    """Pages that no row sees a token of: -1 in the table, NaN in the cache."""
    gone = []
    for s in range(t.seqs):
        first = max(0, int(t.lens[s]) - n[s] + 1 - window) // t.page
        gone += [p for p in t.pages[s, :first] if p >= 0]
        t.pages[s, :first] = -1
    for buf, ref in ((t.k, t.ref.k), (t.v, t.ref.v)):
        ref[gone] = 0x7F
        t.be.upload(buf, ref)
    return len(gone)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("n,window", [([1, 1, 1, 1], 1), ([1, 1, 1, 1], 5), ([1, 1, 1, 1], 100), ([5, 5, 5, 5], 20), ([12, 30, 1, 0], 33),
                                      ([150, 70, 90, 200], 17), ([300, 40, 1, 2], 250)])
def test_pages_before_a_window(be, dtype, page, n, window):
    d = 64 if page < 64 else 128
    t = filled(be, page + window, [700, 517, 130, 1009], 2, page, d)
    assert give_away(t, n, window)
    attend(t, 4, dtype, n, window=window, uniform=len(set(n)) == 1)
    be.synchronize(20000)  # nothing is reported


@pytest.mark.parametrize("page", [16, 64])
def test_a_windowed_sequence_step_by_step(be, page):
    """Single tokens; after each step the pages that fell behind are given away."""
    t = filled(be, 9, [70, 33], 1, page, 64)
    window, desc = 21, ops.HeadDesc(2, 1, 64, 64, ops.F16, ops.NORM_RMS)
    t.width += 10
    t.pages = np.concatenate([t.pages, np.full((2, 10), -1, np.int32)], 1)
    spare, lost = list(set(range(t.ref.k.shape[0])) - set(t.pages.ravel().tolist())), 0
    for step in range(60):
        for s in range(2):
            if t.lens[s] % page == 0:
                t.pages[s, t.lens[s] // page] = spare.pop()
        q, _, _ = append(t, desc, "f16", [1, 1])
        held = t.pages.copy()
        lost += give_away(t, [1, 1], window)
        spare += [p for p in held[held != t.pages]]
        attend(t, 2, "f16", [1, 1], window=window, uniform=step % 2 == 0, q=q.reshape(-1))
        t.check()
        be.synchronize(20000)
    assert lost >= 2
