"""A feed-forward block of the 4-bit operators as a served model runs it: each step
against float64 on its own inputs, then the graph runtime, eager and captured,
against the steps bit for bit."""
import numpy as np
import pytest

import dragonwing_edge_rs_b200 as dw
from dragonwing_edge_rs_b200 import graph as G
from dragonwing_edge_rs_b200 import ops
from tests import _mxfp4_ref as R
from tests.test_gpu_norm import near, norm_tol

pytestmark = pytest.mark.gpu


def operand_values(be, q, s, rows, k):
    return R.values(R.unpack_codes(be.download_array(q, np.uint8), rows, k),
                    R.unpack_scales(be.download_array(s, np.uint8), rows, k), k)


@pytest.mark.parametrize("rows,c,f", [(1, 512, 1400), (37, 200, 333), (130, 1024, 2056), (700, 96, 640)])
def test_block(rows, c, f):
    rng = np.random.default_rng(rows)
    b = G.F16GraphBuilder(3)
    x, r = b.input_f16("x", (rows, c)), b.input_f16("r", (rows, c))
    z, mid = b.mlp_mxfp4(x, r, f, post=ops.NORM_RMS)
    out, y = b.norm_residual(z, mid, post=ops.NORM_LAYER, res_scale=0.5)
    b.g.outputs += [out, y]
    I = b.g.initializers
    n0, up, down, n1 = b.g.ops
    with dw.CudaBackend(0) as be:
        rt = G.CudaGraphRuntime(b.g, be)
        results = []
        for i in range(2):
            xv = rng.normal(0, 1, (rows, c)).astype(np.float16)
            rv = rng.normal(0, 2, (rows, c)).astype(np.float16)
            rt.set_input_bytes("x", xv)
            rt.set_input_bytes("r", rv)
            rt.run()
            got = {t: rt.get_output(t) for t in (mid, z, out, y)}
            x64, r64 = xv.astype(np.float64), rv.astype(np.float64)
            w0, w1 = I[n0.inputs[2]].astype(np.float64), I[n0.inputs[3]].astype(np.float64)
            near(got[mid].astype(np.float64), r64 + R.norm(x64, 1, w0, None, 1e-5),
                 1.01 * (norm_tol(x64, 1, w0, None, 1e-5) + 2.0 ** -24 * np.abs(x64)), "f16")
            # the quantised norm of the stored residual: a value may fall to the other side of a border where its f32
            # lies within the norm's error of one, so all but a few are the definition's own and those are a step off
            m64 = got[mid].astype(np.float64)
            a = operand_values(be, rt.bufs[n0.outputs[1]], rt.bufs[n0.outputs[2]], rows, c)
            a_def = R.values(*R.quantize(R.norm(m64, 1, w1, None, 1e-5)), c)
            assert (a != a_def).mean() < 1e-3 and np.abs(a - a_def).max() <= 0.5 * np.abs(a_def).max()
            # the products, from the operands they had
            wu = R.values(R.unpack_codes(I[up.inputs[2]], f, c), R.unpack_scales(I[up.inputs[3]], f, c), c)
            h = operand_values(be, rt.bufs[up.outputs[0]], rt.bufs[up.outputs[1]], rows, f)
            h_def = R.values(*R.quantize(R.act(a @ wu.T + I[up.inputs[4]], 3)), f)
            assert (h != h_def).mean() < 1e-3 and np.abs(h - h_def).max() <= 0.5 * np.abs(h_def).max()
            wd = R.values(R.unpack_codes(I[down.inputs[2]], c, f), R.unpack_scales(I[down.inputs[3]], c, f), f)
            want = h @ wd.T + I[down.inputs[4]]
            near(got[z].astype(np.float64), want, (f / 16 + 3) * 2.0 ** -23 * (np.abs(h) @ np.abs(wd).T) + 2.0 ** -24 * np.abs(want),
                 "f16")
            z64, wl = got[z].astype(np.float64), I[n1.inputs[2]].astype(np.float64)
            n = R.norm(z64, 2, wl, None, 1e-5)
            near(got[out].astype(np.float64), m64 + 0.5 * n, 0.51 * (norm_tol(z64, 2, wl, None, 1e-5) + 3 * 2.0 ** -24 * np.abs(n)),
                 "f16")
            o64, wp = got[out].astype(np.float64), I[n1.inputs[3]].astype(np.float64)
            near(got[y].astype(np.float64), R.norm(o64, 1, wp, None, 1e-5), norm_tol(o64, 1, wp, None, 1e-5), "f16")
            results.append((xv, rv, got))
        rt.capture()
        for xv, rv, got in results:  # replayed on other inputs: the same bits
            rt.set_input_bytes("x", xv)
            rt.set_input_bytes("r", rv)
            rt.run()
            for t in got:
                np.testing.assert_array_equal(rt.get_output(t).view(np.uint16), got[t].view(np.uint16))
        rt.release()


def test_quantize_ops_in_a_graph():
    b = G.F16GraphBuilder(5)
    x = b.input_f16("x", (9, 70))
    _, n = b.norm_residual(x, None, pre=ops.NORM_LAYER)
    a = b.quantize_mxfp4(n)
    v = b.dequantize_mxfp4(a, 9, 70)
    b.g.outputs.append(v)
    with dw.CudaBackend(0) as be:
        rt = G.CudaGraphRuntime(b.g, be)
        rt.set_input_bytes("x", np.random.default_rng(0).normal(0, 1, (9, 70)).astype(np.float16))
        rt.run()
        nv, got = rt.get_output(n).astype(np.float64), rt.get_output(v).astype(np.float64)
    np.testing.assert_array_equal(got, R.values(*R.quantize(nv), 70))
