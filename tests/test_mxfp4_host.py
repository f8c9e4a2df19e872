"""CPU checks of the MXFP4 format: host quantisation, buffer sizes and scale layout,
and the graph builder's shapes."""
import numpy as np
import pytest

from dragonwing_edge_rs_b200 import graph as G
from dragonwing_edge_rs_b200 import ops
from dragonwing_edge_rs_b200 import quantization as Q
from tests import _mxfp4_ref as R


@pytest.mark.parametrize("rows,k", [(1, 1), (3, 33), (128, 128), (129, 4100), (300, 96)])
def test_host_operand(rows, k):
    rng = np.random.default_rng(k)
    w = (rng.normal(0, 1, (rows, k)) * np.exp(rng.normal(0, 3, (rows, k)))).astype(np.float32)
    w[rng.random(w.shape) < 0.05] = 0
    if k > 32:
        w[rows - 1, 32] = np.nan
        w[0, 0] = -np.inf
    codes, scales = R.quantize(w.astype(np.float64))
    q, s = Q.mxfp4_operand(w)
    assert q.size == ops.mxfp4_code_bytes(rows, k) and s.size == ops.mxfp4_scale_bytes(rows, k)
    np.testing.assert_array_equal(q, R.pack_codes(codes).reshape(-1))
    np.testing.assert_array_equal(s, R.pack_scales(scales, k))


def test_ties_and_values():
    """Every midpoint goes to the even neighbour, and what is decoded is the nearest of the sixteen values."""
    x = np.array([[4.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.9, -0.25, -0.75, -5.0, 6.0, 0.2501, 0.2499]], np.float32)
    q, s = Q.mxfp4_operand(x)
    v = R.values(R.unpack_codes(q, 1, 15), R.unpack_scales(s, 1, 15), 15)
    assert s[0] == 127
    np.testing.assert_array_equal(v[0], [4, 0, 1, 1, 2, 2, 4, 4, 6, 0, -1, -4, 6, 0.5, 0])


def test_scale_tiles_hold_each_place_once():
    at = R.scale_index(300, 500)
    assert len(np.unique(at)) == at.size and at.max() < ops.mxfp4_scale_bytes(300, 500)


def test_builder_shapes_and_work():
    b = G.F16GraphBuilder(1)
    x, r = b.input_f16("x", (5, 96)), b.input_f16("r", (5, 96))
    x, r = b.mlp_mxfp4(x, r, 200)
    out, y = b.norm_residual(x, r)
    g = b.g
    assert g.tensors[out].shape == (5, 96) and g.tensors[y].dtype == "f16"
    assert [o.op_type for o in g.ops] == ["NormResidual", "GemmMxfp4", "GemmMxfp4", "NormResidual"]
    assert g.conv_ops() == 2 * 2 * 5 * 96 * 200
    up = g.ops[1]
    assert g.tensors[up.outputs[0]].nbytes == ops.mxfp4_code_bytes(5, 200)
    assert g.tensors[up.outputs[1]].nbytes == ops.mxfp4_scale_bytes(5, 200)
    assert g.initializers[up.inputs[2]].nbytes == ops.mxfp4_code_bytes(200, 96)
