"""Descriptors that keep buffers' handles: a buffer that is freed is let go, so that a call with the descriptor is
refused (its buffer is null) and reads nothing through the handle that was."""
import ctypes
import gc
import types

import pytest

from dragonwing_edge_rs_b200 import backend as B
from dragonwing_edge_rs_b200 import ops


@pytest.fixture()
def buffers(monkeypatch):
    freed = []
    lib = types.SimpleNamespace(dw_free=lambda be, b: freed.append(b.value) or 0)
    monkeypatch.setattr(B.L, "load", lambda: lib)
    be = types.SimpleNamespace(handle=1, _check=lambda st: None)
    out = [B.CudaBuffer(be, ctypes.c_void_p(4096 + 64 * i), 64) for i in range(4)]
    yield out, freed
    for b in out:
        b.handle = None


def another():  # (of a backend that is closed)
    return B.CudaBuffer(types.SimpleNamespace(handle=None), ctypes.c_void_p(8192), 64)


def test_freed_buffers_leave_their_descriptors(buffers):
    (a, b, c, d), freed = buffers
    heads = [ops.Heads(a, 3, 7), ops.Heads(a)]
    cache, seqs = ops.KvCache(a, b, c, 1, 1, 16, 64), ops.Sequences(b, c, None, 1, 1, 1)
    ragged = ops.Sequences(b, c, d, 1, 1, 1)
    assert [h.buf for h in heads] == [4096, 4096] and (cache.k, cache.v, cache.scales) == (4096, 4160, 4224)
    assert (seqs.table, seqs.lens, seqs.starts, ragged.starts) == (4160, 4224, None, 4288)
    a.free()
    assert [h.buf for h in heads] == [None, None] and cache.k is None and cache.v == 4160 and heads[0].offset == 3
    del heads
    gc.collect()
    b.free(), c.free()
    assert (cache.v, cache.scales, seqs.table, seqs.lens) == (None,) * 4 and ragged.starts == 4288
    assert freed == [4096, 4160, 4224]
    last = ops.Sequences(d, d, d, 1, 1, 1), ops.Sequences(another(), another(), d, 1, 1, 1)
    d.free()  # without its starts a call would take even rows: its table goes, and it is refused
    assert last[0].table is None and last[1].table is None and last[1].lens == 8192
    a.free()  # again: nothing
    assert freed == [4096, 4160, 4224, 4288]


def test_descriptors_made_each_call_do_not_pile_up(buffers):
    (a, *_), _ = buffers
    for _ in range(1000):
        ops.Heads(a)
    gc.collect()
    assert len(a._held) < 200
