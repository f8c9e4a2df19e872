"""A decoder block (attention and feed-forward halves) of the graph runtime, as a served model runs it: a prompt, then
single tokens by a second graph on the same cache; the attention's steps against float64 on their own inputs, captured
replays against eager runs bit for bit."""
import numpy as np
import pytest

import dragonwing_edge_rs_b200 as dw
from dragonwing_edge_rs_b200 import graph as G
from dragonwing_edge_rs_b200 import ops
from tests import _kv_ref as K
from tests.test_gpu_attention import tolerance
from tests.test_gpu_kv_heads import near, rope_tolerance

pytestmark = pytest.mark.gpu


def block(rows, seqs, ragged, c, f, hq, hk, d, page, pages, width, window):
    b = G.F16GraphBuilder(7)
    x, r = b.input_f16("x", (rows, c)), b.input_f16("r", (rows, c))
    cache = b.kv_cache("kv", pages, hk, page, d)
    sq = b.sequences("seq", seqs, width, ragged)
    z, mid = b.attention_mxfp4(x, r, cache, sq, hq, window=window)
    z, mid = b.mlp_mxfp4(z, mid, f, post=ops.NORM_RMS)
    b.g.outputs += [z, mid]
    return b.g


@pytest.mark.parametrize("hq,hk,d,page,window", [(4, 1, 64, 16, 0), (4, 2, 128, 32, 24), (5, 5, 64, 16, 0)])
def test_block(hq, hk, d, page, window):
    c, f, prompts = 192, 320, [50, 7, 21]
    seqs, width = 3, -(-60 // page)
    pages = seqs * width + 1
    rng = np.random.default_rng(d + hq)
    table = rng.permutation(pages)[:seqs * width].reshape(seqs, width).astype(np.int32)
    with dw.CudaBackend(0) as be:
        first = G.CudaGraphRuntime(block(sum(prompts), seqs, True, c, f, hq, hk, d, page, pages, width, window), be)
        kv = {n: first.bufs[n] for n in ("kv_k", "kv_v", "kv_s")}
        after = G.CudaGraphRuntime(block(seqs, seqs, False, c, f, hq, hk, d, page, pages, width, window), be, buffers=kv)
        ref = K.Cache(rng, pages, hk, page, d)
        for n, a in (("kv_k", ref.k), ("kv_v", ref.v), ("kv_s", ref.s)):
            first.set_input_bytes(n, a)
        old = np.zeros(seqs, int)
        for step in range(8):
            rt, n = (first, prompts) if step == 0 else (after, [1] * seqs)
            lens = old + n
            rt.set_input_bytes("seq_table", table)
            rt.set_input_bytes("seq_lens", lens.astype(np.int32))
            starts = np.concatenate([[0], np.cumsum(n)])
            if step == 0:
                rt.set_input_bytes("seq_starts", starts.astype(np.int32))
            for name, size in (("x", 1.0), ("r", 2.0)):
                rt.set_input_bytes(name, rng.normal(0, size, (sum(n), c)).astype(np.float16))
            kinds = {op.op_type: op for op in rt.graph.ops}
            app, att = kinds["AppendKv"], kinds["AttentionKv8"]
            names = [app.inputs[0], app.outputs[0], att.outputs[0], *rt.graph.outputs]
            before = [be.download_array(kv[t], np.uint8) for t in kv]
            rt.run()
            got = {t: rt.get_output(t) for t in names}
            state = [be.download_array(kv[t], np.uint8) for t in kv]
            rows = got[app.inputs[0]].astype(np.float64).reshape(sum(n), -1, d)
            pos = np.concatenate([np.arange(a, b) for a, b in zip(old, lens)])
            freqs = 10000.0 ** (-2.0 * np.arange(d // 2) / d)
            wq, wk = (rt.graph.initializers[app.name + t].astype(np.float64) for t in ("_wq", "_wk"))
            k = K.turn(K.norm(rows[:, hq:hq + hk], 1, wk, 1e-5), pos, freqs, d, False)
            q = K.turn(K.norm(rows[:, :hq], 1, wq, 1e-5), pos, freqs, d, False)
            qg = got[app.outputs[0]].astype(np.float64).reshape(q.shape)
            near(qg, q, rope_tolerance(rows[:, :hq], 1, wq, 1e-5, q, d, False, "f16"))
            for s in range(seqs):
                a, b = starts[s], starts[s + 1]
                ref.append(table[s], int(old[s]), k[a:b], rows[a:b, hq + hk:])
                kk, vv = ref.read(0, table[s], int(lens[s])), ref.read(1, table[s], int(lens[s]))
                want, *how = K.attention(qg[a:b], kk, vv, int(lens[s]), float(np.float32(d ** -0.5)), True, window)
                near(got[att.outputs[0]].astype(np.float64).reshape(qg.shape)[a:b], want, tolerance(want, *how, int(lens[s]), d, "f16"))
            for have, want in zip(state, (ref.k, ref.v, ref.s)):
                np.testing.assert_array_equal(have, want.reshape(-1))
            if step == 2:
                rt.capture()  # from here on steps are replays; this one again
                for t, was in zip(kv, before):
                    be.upload(kv[t], was)
                rt.run()
                for t in names:
                    np.testing.assert_array_equal(rt.get_output(t).view(np.uint16), got[t].view(np.uint16))
                for t, want in zip(kv, state):
                    np.testing.assert_array_equal(be.download_array(kv[t], np.uint8), want)
            old = lens
        for rt in (first, after):
            rt.release()


def test_a_buffer_of_another_size_is_refused():
    g = block(3, 3, False, 64, 64, 2, 1, 64, 16, 4, 1, 0)
    with dw.CudaBackend(0) as be:
        with pytest.raises(dw.BackendError) as e:
            G.CudaGraphRuntime(g, be, buffers={"kv_k": be.alloc(16)})
        assert e.value.status == ops.L.DW_ERR_SIZE_MISMATCH
