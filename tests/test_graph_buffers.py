"""Buffers that a graph is given by name: what needs no GPU."""
import pytest

from dragonwing_edge_rs_b200 import _lib as L
from dragonwing_edge_rs_b200 import graph as G
from dragonwing_edge_rs_b200.backend import BackendError


def test_a_buffer_for_no_tensor_is_refused():
    """A name that the graph does not have, alone or beside one that it has: the graph would run on a buffer of its own."""
    b = G.F16GraphBuilder(1)
    x = b.input_f16("x", (2, 64))
    b.kv_cache("kv", 2, 1, 16, 64)
    b.output_f32(x, "y")
    for buffers in ({"kv_keys": object()}, {"kv_k": object(), "cache_v": object()}):
        with pytest.raises(BackendError) as e:
            G.CudaGraphRuntime(b.g, None, buffers=buffers)
        assert e.value.status == L.DW_ERR_INVALID_ARG and sorted(set(buffers) - {"kv_k"})[0] in e.value.message
