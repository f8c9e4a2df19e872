"""The paged 8-bit cache, what needs no GPU: the reference's own rounding against torch's e4m3, the sizes of the
buffers, how the kernels' work is cut from sequences' rows, and descriptors as the library lays them out."""
import ctypes

import numpy as np
import pytest
import torch

from dragonwing_edge_rs_b200 import _lib as L
from dragonwing_edge_rs_b200 import ops
from tests import _kv_ref as K


def test_reference_rounds_as_e4m3():
    v = np.concatenate([K.VALUES[np.isfinite(K.VALUES)], K.MID, -K.MID, np.random.default_rng(0).normal(0, 100, 20000).clip(-448, 448)])
    # (a float32 that is no exact input would be rounded twice)
    v = v.astype(np.float32).astype(np.float64)
    want = torch.from_numpy(v.astype(np.float32)).to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    np.testing.assert_array_equal(K.codes(v), want)
    back = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).float().numpy()
    np.testing.assert_array_equal(K.VALUES.astype(np.float32), back)


def test_reference_exponent():
    for e in (-64, -63, 0, 5, 63):
        assert K.exponent(448.0 * 2.0 ** e) == e
        assert K.exponent(np.nextafter(448.0 * 2.0 ** e, np.inf)) == min(e + 1, 63)
    assert K.exponent(0.0) == -64 and K.exponent(1e30) == 63


def test_sizes():
    assert ops.kv_code_bytes(10, 3, 16, 64) == 10 * 3 * 16 * 64
    assert ops.kv_scale_bytes(10, 3) == 60


def test_no_backend_is_an_error():
    lib = L.load()
    out = ctypes.c_void_p()
    f = (ctypes.c_double * 1)(1.0)
    assert lib.dw_prepare_rope(None, f, 1, ctypes.byref(out)) == L.DW_ERR_INVALID_ARG
    assert lib.dw_norm_rope(None, None, 1, *[None] * 8) == L.DW_ERR_INVALID_ARG
    assert lib.dw_append_kv(None, *[None] * 10) == L.DW_ERR_INVALID_ARG
    assert lib.dw_read_kv(None, None, None, 0, None, None) == L.DW_ERR_INVALID_ARG
    assert lib.dw_attention_kv8(None, *[None] * 5) == L.DW_ERR_INVALID_ARG


@pytest.mark.parametrize("per,size,extra", [(1, 16, 2), (1, 128, 2), (4, 16, 1), (5, 16, 1), (1, 1, 0), (7, 256, 1)])
def test_items_cover_every_row(per, size, extra):
    """The rule of seq_items / seq_of_item (csrc/dw_kv.cuh), followed on the host: every block of rows, and every
    page that rows lie in, is some launched item's."""
    rng = np.random.default_rng(per * size)
    for trial in range(60):
        seqs = int(rng.integers(1, 70))
        n = rng.choice([0, 0, 1, 1, 2, 15, 16, 17, 300], seqs) if trial else np.ones(seqs, np.int64)
        starts = np.concatenate([[0], np.cumsum(n)])
        tokens = int(starts[-1]) + int(rng.integers(0, 5))
        if not tokens:
            continue
        first = starts[:-1] * per // size + extra * np.arange(seqs)

        def of_item(w):
            lo, count = 0, seqs
            while count > 1:
                step = (count + 31) // 32
                at = np.arange(32) * step
                ok = [j for j in range(32) if at[j] < count and first[lo + at[j]] <= w]
                k = max(ok + [0])
                lo, count = lo + k * step, min(step, count - k * step)
            return lo, w - first[lo]

        got = {}
        for w in range(tokens * per // size + extra * seqs):
            s, place = of_item(w)
            if place >= 0:
                got.setdefault(s, set()).add(place)
        for s in range(seqs):
            blocks = -(-int(n[s]) * per // size)
            if extra == 2:  # pages: the rows may begin anywhere in their first
                blocks = max(((int(n[s]) + o - 1) // size + 1) for o in range(size)) if n[s] else 0
            assert set(range(blocks)) <= got.get(s, set()), (s, n[s])
