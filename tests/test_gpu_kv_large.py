"""The paged 8-bit cache where offsets pass 32 bits: pages behind the first 4 GiB of codes, and a long sequence."""
import numpy as np
import pytest
import torch

import dragonwing_edge_rs_b200 as dw
from dragonwing_edge_rs_b200 import ops
from tests import _kv_ref as K
from tests.test_gpu_attention import tolerance

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n", [1, 100])
def test_pages_behind_four_gigabytes(n):
    pages, hk, page, d, hq = 36000, 8, 128, 128, 8  # 4.7 GB of codes each
    rng = np.random.default_rng(n)
    free, _ = torch.cuda.mem_get_info()
    if free < 14 << 30:
        pytest.skip("needs 14 GB of device memory")
    with dw.CudaBackend(0) as be:
        k, v = be.alloc(ops.kv_code_bytes(pages, hk, page, d)), be.alloc(ops.kv_code_bytes(pages, hk, page, d))
        s = be.alloc(ops.kv_scale_bytes(pages, hk))
        cache = ops.KvCache(k, v, s, pages, hk, page, d)
        table = np.array([[pages - 1, 3, pages - 2, 34999]], np.int32)
        length = 400
        up = be.upload_array
        desc = ops.HeadDesc(hq, hk, d, 0, ops.F32, 0)
        seqs = ops.Sequences(up(table), up(np.array([length], np.int32)), None, 1, length, 4)
        x = rng.normal(0, 1, (length, 2 * hk * d)).astype(np.float32)
        buf = up(x)
        ops.append_kv(be, desc, cache, seqs, ops.Heads(buf, 0, 2 * hk * d), ops.Heads(buf, hk * d, 2 * hk * d))
        ref = K.Cache(rng, 4, hk, page, d)
        rows = x.astype(np.float64).reshape(length, 2 * hk, d)
        ref.append(np.arange(4), 0, rows[:, :hk], rows[:, hk:])
        out = [be.alloc(length * hk * d * 4) for _ in range(2)]
        ops.read_kv(be, cache, seqs, ops.F32, ops.Heads(out[0]), ops.Heads(out[1]))
        kk, vv = ref.read(0, np.arange(4), length), ref.read(1, np.arange(4), length)
        np.testing.assert_array_equal(be.download_array(out[0], np.float32), kk.reshape(-1))
        np.testing.assert_array_equal(be.download_array(out[1], np.float32), vv.reshape(-1))
        q = rng.normal(0, 1, (n, hq, d)).astype(np.float16)
        y = be.alloc(q.nbytes)
        ops.attention_kv8(be, ops.AttentionDesc(hq, ops.F16, d ** -0.5), cache,
                          ops.Sequences(seqs.keep[0], seqs.keep[1], None, 1, n, 4), ops.Heads(up(q)), ops.Heads(y))
        want, *how = K.attention(q.astype(np.float64), kk, vv, length, float(np.float32(d ** -0.5)), True, 0)
        got = be.download_array(y, np.float16).astype(np.float64).reshape(want.shape)
        assert (np.abs(got - want) <= tolerance(want, *how, length, d, "f16")).all()


def test_a_long_sequence():
    """300000 tokens, every one a sum's part: against float64 in torch on the values that the cache gives back."""
    hk, page, d, hq, length = 1, 64, 128, 4, 300000
    width = -(-length // page)
    g = torch.Generator(device="cuda").manual_seed(1)
    with dw.CudaBackend(0) as be:
        k, v = be.alloc(ops.kv_code_bytes(width, hk, page, d)), be.alloc(ops.kv_code_bytes(width, hk, page, d))
        s = be.alloc(ops.kv_scale_bytes(width, hk))
        cache = ops.KvCache(k, v, s, width, hk, page, d)
        up = be.upload_array
        table, lens = up(np.random.default_rng(0).permutation(width).astype(np.int32)), up(np.array([length], np.int32))
        x = torch.randn(length, 2 * d, generator=g, device="cuda").half()
        torch.cuda.synchronize()
        buf = be.wrap(x.data_ptr(), x.numel() * 2)
        whole = ops.Sequences(table, lens, None, 1, length, width)
        ops.append_kv(be, ops.HeadDesc(hq, hk, d, 0, ops.F16, 0), cache, whole, ops.Heads(buf, 0, 2 * d), ops.Heads(buf, d, 2 * d))
        kv = torch.empty(2, length, d, device="cuda")
        bufs = [be.wrap(t.data_ptr(), t.numel() * 4) for t in kv]
        ops.read_kv(be, cache, whole, ops.F32, ops.Heads(bufs[0]), ops.Heads(bufs[1]))
        be.synchronize()
        for n in (1, 40):
            q = torch.randn(n, hq, d, generator=g, device="cuda").half()
            y = torch.empty_like(q)
            torch.cuda.synchronize()
            wrap = lambda t: ops.Heads(be.wrap(t.data_ptr(), t.numel() * 2))
            ops.attention_kv8(be, ops.AttentionDesc(hq, ops.F16, d ** -0.5), cache, ops.Sequences(table, lens, None, 1, n, width), wrap(q), wrap(y))
            be.synchronize()
            k64, v64 = kv.double()
            t = (q.double().view(-1, d) @ k64.T).view(n, hq, length) * float(np.float32(d ** -0.5))
            pos = torch.arange(length - n, length, device="cuda")[:, None, None]
            t = t.masked_fill(torch.arange(length, device="cuda") > pos, -np.inf)
            w = torch.softmax(t, -1)
            want, mean = w @ v64, w @ v64.abs()
            mass = (q.double().abs().view(-1, d) @ k64.abs().T).view(n, hq, length).amax(-1, keepdim=True) * d ** -0.5
            big = t.masked_fill(t == -np.inf, 0).abs().amax(-1, keepdim=True)
            tol = tolerance(*(a.cpu().numpy() for a in (want, mean, big, mass)), length, d, "f16")
            assert (np.abs(y.double().cpu().numpy() - want.cpu().numpy()) <= tol).all()
