"""How calls over sequences are cut into items of work, by the library's own rule (the kernels' search, on the host):
every block of a sequence's rows, and every page that its rows lie in, is some launched item's, and no two items are
the same."""
import ctypes

import numpy as np
import pytest

from dragonwing_edge_rs_b200 import _lib as L


def items(starts, seqs, tokens, per, size, extra):
    lib = L.load()
    at = None if starts is None else starts.ctypes.data
    n = lib.dw_debug_seq_items(at, seqs, tokens, per, size, extra, None, None)
    seq, place = np.empty(n, np.uint32), np.empty(n, np.int64)
    assert lib.dw_debug_seq_items(at, seqs, tokens, per, size, extra, seq.ctypes.data, place.ctypes.data) == n
    return seq, place


def blocks(n, per, size, extra):
    """Of a sequence's n rows at most."""
    if extra == 2:  # pages: the rows may begin anywhere in their first
        return max((n + o - 1) // size + 1 for o in range(size)) if n else 0
    return -(-n * per // size)


RULES = [(1, 16, 2), (1, 32, 2), (1, 128, 2), (4, 8, 1), (4, 16, 1), (5, 24, 1), (1, 1, 0), (7, 256, 1), (33, 256, 1)]


def covered(seq, place, n, rule):
    for s in range(len(n)):
        mine = place[seq == s]
        assert set(range(blocks(int(n[s]), *rule))) <= set(mine.tolist()), (s, n[s])
    pairs = np.stack([seq, place])
    assert len(np.unique(pairs, axis=1).T) == len(seq)


@pytest.mark.parametrize("rule", RULES)
def test_ragged(rule):
    rng = np.random.default_rng(rule[0] * rule[1])
    for trial in range(60):
        seqs = int(rng.choice([1, 2, 31, 32, 33, 70, 1025]))
        n = rng.choice([0, 0, 1, 1, 2, 15, 16, 17, 300], seqs) if trial else np.ones(seqs, np.int64)
        first = int(rng.integers(0, 4))  # rows of no sequence in front and behind
        starts = (first + np.concatenate([[0], np.cumsum(n)])).astype(np.int32)
        tokens = int(starts[-1]) + int(rng.integers(0, 5))
        if tokens:
            covered(*items(starts, seqs, tokens, *rule), n, rule)


@pytest.mark.parametrize("rule", RULES)
@pytest.mark.parametrize("n", [1, 2, 15, 16, 17, 129, 300])
@pytest.mark.parametrize("seqs", [1, 3, 64])
def test_even(rule, n, seqs):
    covered(*items(None, seqs, n * seqs, *rule), np.full(seqs, n), rule)


def test_starts_beyond_32_bits_of_items():
    """Offsets of rows times heads pass 32 bits."""
    starts = np.array([0, 2 ** 31 - 10, 2 ** 31 - 2], np.int32)
    lib = L.load()
    n = lib.dw_debug_seq_items(starts.ctypes.data, 2, 2 ** 31 - 1, 4, 256, 1, None, None)
    assert n == (2 ** 31 - 1) * 4 // 256 + 2
    assert lib.dw_debug_seq_items(starts.ctypes.data, 0, 5, 1, 16, 1, None, None) == 0
    assert lib.dw_debug_seq_items(ctypes.c_void_p(), 2, 6, 1, 0, 1, None, None) == 0
