"""Graphs that change state: capturing one runs nothing."""
import ctypes

import numpy as np
import pytest

import dragonwing_edge_rs_b200 as dw
from dragonwing_edge_rs_b200 import graph as G
from dragonwing_edge_rs_b200 import ops
from tests.test_gpu_attention_block import block

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("before", ["unset", "old"])
def test_capture_leaves_the_cache_and_outputs_alone(before):
    """Before any length is set, and with those of the step before."""
    seqs, page, pages, width = 3, 16, 10, 3
    rng = np.random.default_rng(1)
    with dw.CudaBackend(0) as be:
        rt = G.CudaGraphRuntime(block(seqs, seqs, False, 128, 192, 4, 2, 64, page, pages, width, 0), be)
        kept = ["kv_k", "kv_v", "kv_s", *rt.graph.outputs]
        for n in kept:
            rt.set_input_bytes(n, rng.integers(0, 120, rt.graph.tensors[n].nbytes).astype(np.uint8))
        lens = np.full(seqs, 1 << 30 if before == "unset" else 20, np.int32)  # (what a buffer may hold that nobody set)
        rt.set_input_bytes("seq_table", np.arange(seqs * width, dtype=np.int32))
        rt.set_input_bytes("seq_lens", lens)
        for n in ("x", "r"):
            rt.set_input_bytes(n, rng.normal(0, 1, (seqs, 128)).astype(np.float16))
        held, launches = [rt.get_output_bytes(n) for n in kept], be.launch_count()
        kernels = rt.capture()
        be.synchronize(20000)
        assert be.launch_count() == launches
        for n, want in zip(kept, held):
            np.testing.assert_array_equal(rt.get_output_bytes(n), want)
        rt.set_input_bytes("seq_lens", np.full(seqs, 21, np.int32))
        rt.run()
        be.synchronize(20000)
        assert be.launch_count() - launches == kernels >= len(rt.graph.ops)
        got = [rt.get_output_bytes(n) for n in kept]
        assert rt.capture() == kernels  # again: the one before is let go
        for n, want in zip(kept[:3], held):
            rt.set_input_bytes(n, want)
        rt.run()
        for n, want in zip(kept, got):
            np.testing.assert_array_equal(rt.get_output_bytes(n), want)
        rt.release()


def test_kernels_of_a_graph():
    lib = ops.L.load()
    assert lib.dw_graph_kernels(None) == 0
    with dw.CudaBackend(0) as be:
        x, y = be.upload_array(np.zeros(64, np.float16)), be.alloc(256)
        g = ctypes.c_void_p()
        be._check(lib.dw_capture_begin(be.handle))
        for _ in range(3):
            ops.cast_f16_to_f32(be, x, y)
        be._check(lib.dw_capture_end(be.handle, ctypes.byref(g)))
        assert lib.dw_graph_kernels(g) == 3
        lib.dw_graph_destroy(g)
