"""The attention half of a served transformer block, as cases to measure: norms of the query and key heads with
the position rotation, appending keys and values to a paged cache held in 8 bits, attention over that cache, and
the run of them that a layer makes.

Rows are tokens; a row holds heads one after the other, each of d values.  The packed rows of a projection hold
the query heads, then the key heads, then the value heads.

Sequence s has `lens[s]` tokens in the cache, the rows' own among them: its n rows are the positions
lens[s] - n .. lens[s] - 1.  `table[s]` names the pages that hold its tokens, `page` tokens each.

The cache: pages [pages, kv heads, page, d] of e4m3 codes, for keys and for values, and for each page and head
two scale bytes (keys, values), e + 127 for the scale X = 2^e.  A value is held as the e4m3 nearest to v / X
(ties to even).  X is the smallest power of two, 2^-64 to 2^63, with max|v| <= 448 X over the block, and never
below the X that tokens already held in the block have; where it grows, their codes are rounded again.

Rotation: pair i of a head (elements i and i + rot / 2, or 2 i and 2 i + 1) turns by position * freqs[i].

Attention: query row i at position p sees the keys at 0 .. p (with a window w: p - w + 1 .. p) of its sequence,
softmax(scale * q k) v in the head's group.

`run` computes each operator in elementary torch operations, or with `own` by this repository's entry points;
`exact` computes the definition in 64 bits.
"""
import math

import torch

own = False

_TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_SIZE = {"f32": 4, "f16": 2, "bf16": 2}
_EPS = 1e-5
_backend = None


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------

def _rope(name, tokens, hq, hk, d, type, rot=None, pairs="halves", norm="rms", far=0):
    return {"name": name, "op": "rope", "tokens": tokens, "hq": hq, "hk": hk, "d": d, "rot": d if rot is None else rot, "pairs": pairs,
            "norm": norm, "far": far, "type": type}


def _cache(name, op, seqs, new, old, hq, hk, d, page, type, ragged=False, window=0, norm="rms"):
    return {"name": name, "op": op, "seqs": seqs, "new": new, "old": old, "hq": hq, "hk": hk, "d": d, "page": page, "type": type,
            "ragged": ragged, "window": window, "norm": norm}


def listed():
    return [
        # the query and key heads of a long prompt
        _rope("rope prompt", 8192, 32, 8, 128, "bf16"),
        # those of a single token
        _rope("rope token", 1, 32, 8, 128, "f16"),
        # half of each head turned, neighbouring pairs, at far positions, in f32
        _rope("rope far", 333, 12, 3, 64, "f32", rot=32, pairs="neighbours", norm="layer", far=1 << 20),
        # a prompt's keys and values into an empty cache, its queries on the way
        _cache("append prompt", "append", 1, 4096, 0, 32, 8, 128, 64, "bf16"),
        # one token for each sequence of a batch, into pages that hold others
        _cache("append batch", "append", 64, 1, 1000, 32, 8, 128, 16, "f16", ragged=True),
        # a single token that looks back over a conversation
        _cache("attend token", "attend", 1, 1, 4000, 32, 8, 128, 64, "f16"),
        # one token for each sequence of a large batch, lengths from short to 8192
        _cache("attend batch", "attend", 64, 1, 8191, 32, 8, 128, 64, "bf16", ragged=True),
        # five drafted tokens to verify for each sequence
        _cache("attend drafts", "attend", 16, 5, 4000, 32, 8, 128, 32, "bf16", ragged=True),
        # a long prompt
        _cache("attend prompt", "attend", 1, 4096, 0, 32, 8, 128, 64, "bf16"),
        # pieces of prompts behind what is cached, in a window, odd groups of small heads
        _cache("attend pieces", "attend", 3, 700, 5000, 20, 4, 64, 16, "f16", ragged=True, window=1000),
        # a layer's attention for one token of each sequence
        _cache("layer batch", "layer", 32, 1, 2000, 32, 8, 128, 64, "f16", ragged=True),
        # and for two prompts
        _cache("layer prompt", "layer", 2, 1500, 0, 32, 8, 128, 64, "bf16", ragged=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rope", "append", "attend", "attend", "layer"])
    d, t = rng.choice([64, 128]), rng.choice(["f16", "bf16"])
    hk = rng.choice([1, 2, 3, 4, 8])
    hq = hk * rng.choice([1, 2, 4, 5, 8])
    if op == "rope":
        tokens = max(1, min(_log(rng, 1, 8192), 8192 * 40 * 128 // ((hq + hk) * d)))
        c = _rope("", tokens, hq, hk, d, rng.choice(["f32", "f16", "bf16"]), rot=rng.choice([d, d, d // 2]),
                  pairs=rng.choice(["halves", "neighbours"]), norm=rng.choice(["rms", "none", "layer"]), far=rng.choice([0, 1 << 17]))
        if c["type"] == "f32":
            c["tokens"] = max(1, tokens // 2)
    else:
        seqs = _log(rng, 1, 64)
        if rng.random() < 0.6:  # a few tokens for each sequence
            new, old = rng.choice([1, 1, 2, 4, 7]), _log(rng, 1, 8000)
            old = min(old, 64 * 8000 * 8 * 128 // (seqs * hk * d * new))
        else:                   # prompts and pieces of them
            seqs = min(seqs, 8)
            new = max(1, _log(rng, 16, 4096) // seqs)
            old = rng.choice([0, 0, _log(rng, 1, 4000) // seqs])
        c = _cache("", op, seqs, new, old, hq, hk, d, rng.choice([16, 32, 64, 128]), t, ragged=rng.random() < 0.6,
                   window=rng.choice([0, 0, _log(rng, 16, 4000)]) if op != "append" else 0, norm=rng.choice(["rms", "none"]))
    del c["name"]
    return c


def _spread(n, most, ragged, phase):
    """n whole numbers up to `most`, spread evenly over 1 .. most where ragged."""
    if not ragged:
        return [most] * n
    return [min(most, 1 + int(most * math.modf((i + phase) * 0.6180339887498949)[0])) for i in range(n)]


def _plan(c):
    """(rows, length) of each sequence."""
    new = _spread(c["seqs"], c["new"], c["ragged"] and c["new"] > 16, 1)  # a step adds as many tokens to each
    old = _spread(c["seqs"], c["old"], c["ragged"], 2) if c["old"] else [0] * c["seqs"]
    return [(n, n + o) for n, o in zip(new, old)]


def _touched(c, plan):
    """The tokens of each sequence that lie in pages which its rows are written to."""
    return [length - (length - n) // c["page"] * c["page"] for n, length in plan]


def _seen(c, plan):
    """(key-query pairs, keys seen by any query) of all sequences, for one head."""
    pairs = keys = 0
    for n, length in plan:
        w = c["window"] or length
        full = max(0, min(n, length - w + 1))  # rows whose window is full
        short = n - full
        pairs += full * w + short * (length - n + 1) + short * (short - 1) // 2
        keys += min(length, n + w - 1)
    return pairs, keys


def work(case):
    c = case
    hq, hk, d, es = c["hq"], c["hk"], c["d"], _SIZE[c["type"]]
    if c["op"] == "rope":
        n = c["tokens"] * (hq + hk) * d
        return {"bytes": 2 * n * es + 4 * c["tokens"] + 8 * d, "flops": 9 * n}
    plan = _plan(c)
    tokens = sum(n for n, _ in plan)
    pairs, keys = _seen(c, plan)
    # rows in, queries out, codes out; the pages that were touched in and their values out
    append = tokens * (2 * hq + 2 * hk) * d * es + tokens * hk * d * 2
    touched = sum(_touched(c, plan)) * hk * d * 2 * (1 + es)
    attend = 2 * tokens * hq * d * es + keys * hk * d * 2
    flops = 4.0 * pairs * hq * d
    if c["op"] == "append":
        return {"bytes": append + touched, "flops": 9 * tokens * (hq + 2 * hk) * d}
    if c["op"] == "attend":
        return {"bytes": attend, "flops": flops}
    return {"bytes": append + attend + touched, "flops": flops + 9 * tokens * (hq + 2 * hk) * d}


# ---------------------------------------------------------------------------
# the cache in torch
# ---------------------------------------------------------------------------

def _pow2(e):
    """2^e for whole e, exactly, in f64."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _scale_exponent(amax):
    """The smallest e in -64 .. 63 with amax <= 448 * 2^e; amax f64."""
    m, x = torch.frexp(amax)  # amax = m * 2^x, m in [0.5, 1); 448 = 0.875 * 2^9
    return torch.where(amax > 0, x.long() - 9 + (m > 0.875), -64).clamp(-64, 63)


def _e4m3(v):
    """v f64 rounded to the nearest e4m3 value, ties to even, 448 at most."""
    a = v.abs()
    step = _pow2((torch.frexp(a)[1].long() - 1).clamp(min=-6) - 3)
    return torch.copysign((torch.round(a / step) * step).clamp(max=448.0), v)


def _codes(v):
    """e4m3 values -> their codes."""
    return v.to(torch.float32).to(torch.float8_e4m3fn).view(torch.uint8)


def _decoded(codes):
    return codes.view(torch.float8_e4m3fn).to(torch.float32)


def _read(s, which, table, length):
    """The values of the first `length` tokens of a sequence, f32 [length, hk, d]."""
    pages = table[:-(-length // s["case"]["page"])].long()
    x = _pow2(s["scales"][pages, :, "kv".index(which)].long() - 127).float()[:, :, None, None]
    return (_decoded(s[which][pages]) * x).transpose(1, 2).flatten(0, 1)[:length]


# ---------------------------------------------------------------------------
# states
# ---------------------------------------------------------------------------

def _freqs(rot):
    return [10000.0 ** (-2.0 * i / rot) for i in range(rot // 2)]


def _heads(g, rows, heads, d):
    """Rows of heads as projections give them: normal, heads and channels of different size."""
    size = torch.exp(0.5 * torch.randn(heads, 1, generator=g, device="cuda") + 0.5 * torch.randn(heads, d, generator=g, device="cuda"))
    return torch.randn(rows, heads, d, generator=g, device="cuda") * size


def prepare(case, seed):
    c = case
    if own:
        _open()
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    dev, t = "cuda", _TYPES[c["type"]]
    hq, hk, d = c["hq"], c["hk"], c["d"]
    s = {"case": c}
    s["wq"] = 1.0 + 0.2 * torch.randn(d, generator=g, device=dev)
    s["wk"] = 1.0 + 0.2 * torch.randn(d, generator=g, device=dev)
    if c["op"] == "rope":
        n = c["tokens"]
        s["x"] = _heads(g, n, hq + 2 * hk, d).to(t).flatten(1)
        s["pos"] = (torch.arange(n, device=dev) + torch.randint(0, c["far"] + 1, (n,), generator=g, device=dev)).int()
        s["q"], s["y"] = torch.empty(n, hq * d, dtype=t, device=dev), torch.empty(n, hk * d, dtype=t, device=dev)
        if own:
            _wrap(s)
        return s
    page = c["page"]
    s["plan"] = plan = _plan(c)
    rows = sum(n for n, _ in plan)
    need = [-(-length // page) for _, length in plan]
    pages, width = sum(need) + 3, max(need)
    order = torch.randperm(pages, generator=g, device=dev).int()
    s["table"] = torch.full((c["seqs"], width), -1, dtype=torch.int32, device=dev)
    at = 0
    for i, n in enumerate(need):
        s["table"][i, :n] = order[at:at + n]
        at += n

    def column(v):
        return torch.tensor(v, dtype=torch.int32, device=dev)

    def starts(counts):
        return column([sum(counts[:i]) for i in range(len(counts) + 1)])

    s["lens"] = column([length for _, length in plan])
    s["starts"] = starts([n for n, _ in plan])
    # what the pages hold: tokens as an append left them (in pages that no token was written to yet, anything that
    # an earlier owner left)
    for which in "kv":
        s[which] = torch.empty(pages, hk, page, d, dtype=torch.uint8, device=dev)
    s["scales"] = torch.empty(pages, hk, 2, dtype=torch.uint8, device=dev)
    size = torch.exp(0.5 * torch.randn(hk, 1, d, generator=g, device=dev))
    for a in range(0, pages, 512):
        b = min(pages, a + 512)
        for i, which in enumerate("kv"):
            v = torch.randn(b - a, hk, page, d, generator=g, device=dev) * size
            e = _scale_exponent(v.abs().flatten(2).amax(-1).double())
            s[which][a:b] = (v / _pow2(e).float()[:, :, None, None]).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
            s["scales"][a:b, :, i] = (e + 127).to(torch.uint8)
    if c["op"] == "attend":
        s["x"] = (torch.randn(rows, hq * d, generator=g, device=dev) * 1.5).to(t)
        s["o"] = torch.empty(rows, hq * d, dtype=t, device=dev)
    else:
        s["x"] = _heads(g, rows, hq + 2 * hk, d).to(t).flatten(1)
        s["q"] = torch.empty(rows, hq * d, dtype=t, device=dev)
        if c["op"] == "layer":
            s["o"] = torch.empty(rows, hq * d, dtype=t, device=dev)
        s["touched"] = touched = _touched(c, plan)
        s["t_starts"] = starts(touched)
        s["kt"] = torch.empty(sum(touched), hk * d, dtype=t, device=dev)
        s["vt"] = torch.empty(sum(touched), hk * d, dtype=t, device=dev)
    if own:
        _wrap(s)
    return s


def _open():
    """The backend, with its stream as torch's current one: inputs are made before the operators read them, and
    what torch does with the outputs comes after them."""
    global _backend
    import dragonwing_edge_rs_b200 as dw
    if _backend is None:
        _backend = dw.CudaBackend(torch.cuda.current_device())
    torch.cuda.set_stream(torch.cuda.ExternalStream(_backend.stream()))


def _wrap(s):
    """A program of the framework holds its data in the backend's buffers, and its descriptors: the same memory,
    wrapped once."""
    from dragonwing_edge_rs_b200 import ops
    be, c = _backend, s["case"]
    b = {n: be.wrap(t.data_ptr(), t.numel() * t.element_size()) for n, t in s.items() if isinstance(t, torch.Tensor)}
    t = {"f32": ops.F32, "f16": ops.F16, "bf16": ops.BF16}[c["type"]]
    hq, hk, d = c["hq"], c["hk"], c["d"]
    kinds = {"none": ops.NORM_NONE, "rms": ops.NORM_RMS, "layer": ops.NORM_LAYER}
    s["b"], s["t"] = b, t
    rot = c.get("rot", d)
    s["heads"] = ops.HeadDesc(hq, hk, d, rot, t, kinds[c["norm"]], _EPS, c.get("pairs") == "neighbours")
    s["freqs"] = ops.prepare_rope(be, _freqs(rot))
    if c["op"] != "attend":
        width = (hq + 2 * hk) * d
        s["qkv"] = [ops.Heads(b["x"], o * d, width) for o in (0, hq, hq + hk)]
        s["q_out"] = ops.Heads(b["q"])
    if c["op"] == "rope":
        s["k_out"] = ops.Heads(b["y"])
        return
    s["cache"] = ops.KvCache(b["k"], b["v"], b["scales"], s["k"].shape[0], hk, c["page"], d)

    def sequences(starts, rows):
        return ops.Sequences(b["table"], b["lens"], starts, c["seqs"], rows, s["table"].shape[1])

    same = all(n == s["plan"][0][0] for n, _ in s["plan"])
    s["seq"] = sequences(None if same else b["starts"], s["x"].shape[0])
    if c["op"] != "attend":
        s["t_seq"] = sequences(b["t_starts"], s["kt"].shape[0])
        s["k_read"], s["v_read"] = ops.Heads(b["kt"]), ops.Heads(b["vt"])
    if c["op"] != "append":
        s["attend"] = ops.AttentionDesc(hq, t, 1.0 / math.sqrt(d), True, c["window"])
        s["att_q"], s["att_o"] = ops.Heads(b["x"] if c["op"] == "attend" else b["q"]), ops.Heads(b["o"])


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------

def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(s):
    from dragonwing_edge_rs_b200 import ops
    be, b, c = _backend, s["b"], s["case"]
    if c["op"] == "rope":
        q, k, _ = s["qkv"]
        ops.norm_rope(be, s["heads"], c["tokens"], q, k, b["wq"], b["wk"], s["freqs"], b["pos"], s["q_out"], s["k_out"])
        return s["q"], s["y"]
    if c["op"] != "attend":
        q, k, v = s["qkv"]
        ops.append_kv(be, s["heads"], s["cache"], s["seq"], k, v, b["wk"], s["freqs"], q, b["wq"], s["q_out"])
    if c["op"] != "append":
        ops.attention_kv8(be, s["attend"], s["cache"], s["seq"], s["att_q"], s["att_o"])
    if c["op"] == "attend":
        return s["o"]
    ops.read_kv(be, s["cache"], s["t_seq"], s["t"], s["k_read"], s["v_read"])
    return (s["q"] if c["op"] == "append" else s["o"]), s["kt"], s["vt"]


def _norm(x, kind, w):
    if kind == "none":
        return x
    if kind == "layer":
        x = x - x.mean(-1, keepdim=True)
    return x / torch.sqrt((x * x).mean(-1, keepdim=True) + _EPS) * w.to(x.dtype)


def _turned(x, pos, rot, neighbours):
    """x [rows, heads, d] in 32 or 64 bits, turned; angles in 64 bits."""
    f = torch.tensor(_freqs(rot), dtype=torch.float64, device=x.device)
    a = pos.double()[:, None, None] * f
    cos, sin = torch.cos(a).to(x.dtype), torch.sin(a).to(x.dtype)
    if neighbours:
        u, v = x[..., 0:rot:2], x[..., 1:rot:2]
        y = torch.stack((u * cos - v * sin, u * sin + v * cos), -1).flatten(-2)
    else:
        u, v = x[..., :rot // 2], x[..., rot // 2:rot]
        y = torch.cat((u * cos - v * sin, u * sin + v * cos), -1)
    return torch.cat((y, x[..., rot:]), -1)


def _append_plain(s):
    c = s["case"]
    hq, hk, d, page = c["hq"], c["hk"], c["d"], c["page"]
    rows = s["x"].shape[0]
    x = s["x"].view(rows, -1, d)
    pos = torch.cat([torch.arange(length - n, length, device=x.device) for n, length in s["plan"]])
    q = _turned(_norm(x[:, :hq].float(), c["norm"], s["wq"]), pos, d, False).to(x.dtype)
    # what a value next to a border of its 8 bits becomes hangs on its last bits: 64 of them
    k = _turned(_norm(x[:, hq:hq + hk].double(), c["norm"], s["wk"]), pos, d, False)
    v = x[:, hq + hk:].double()
    at = 0
    for i, (n, length) in enumerate(s["plan"]):
        old = length - n
        first, last = old // page, (length - 1) // page
        ids = s["table"][i, first:last + 1].long()
        head = old - first * page  # tokens that the first page holds
        for j, (which, u) in enumerate((("k", k), ("v", v))):
            e_old = s["scales"][ids, :, j].long() - 127
            new = torch.zeros((last - first + 1) * page, hk, d, dtype=torch.float64, device=x.device)
            new[head:head + n] = u[at:at + n]
            new = new.view(-1, page, hk, d).transpose(1, 2)
            e = _scale_exponent(new.abs().amax((2, 3)))
            if head:
                e[0] = torch.maximum(e[0], e_old[0])
            codes = _codes(_e4m3(new / _pow2(e)[:, :, None, None]))
            if head:
                was = _decoded(s[which][ids[0], :, :head]).double() * _pow2(e_old[0] - e[0])[:, None, None]
                codes[0, :, :head] = _codes(_e4m3(was))
            tail = length - last * page  # places behind the last token keep what they hold
            codes[-1, :, tail:] = s[which][ids[-1], :, tail:]
            s[which][ids] = codes
            s["scales"][ids, :, j] = (e + 127).to(torch.uint8)
        at += n
    return q.flatten(1)


def _touched_plain(s):
    out = []
    for which in "kv":
        parts = [_read(s, which, s["table"][i], length)[length - n:] for i, (n, (_, length)) in enumerate(zip(s["touched"], s["plan"]))]
        out.append(torch.cat(parts).flatten(1).to(s["x"].dtype))
    return out


def _attend_plain(s, q):
    c = s["case"]
    hq, hk, d = c["hq"], c["hk"], c["d"]
    out, at = [], 0
    for i, (n, length) in enumerate(s["plan"]):
        k, v = _read(s, "k", s["table"][i], length), _read(s, "v", s["table"][i], length)
        first = max(0, length - n - c["window"] + 1) if c["window"] else 0  # no row sees an earlier key
        k, v = k[first:].permute(1, 2, 0), v[first:].transpose(0, 1)
        qi = q[at:at + n].view(n, hk, hq // hk, d).float().permute(1, 2, 0, 3)
        pos = torch.arange(length - n, length, device=q.device)[:, None]
        key = torch.arange(first, length, device=q.device)[None]
        hidden = (key > pos) | (key <= pos - c["window"]) if c["window"] else key > pos
        o = torch.empty(n, hk, hq // hk, d, device=q.device)
        for h in range(hk):
            logits = (qi[h].reshape(-1, d) @ k[h]).view(hq // hk, n, -1) * (1.0 / math.sqrt(d))
            logits = logits.masked_fill(hidden, -math.inf)
            p = torch.exp(logits - logits.amax(-1, keepdim=True))
            o[:, h] = ((p.view(-1, p.shape[-1]) @ v[h]).view(hq // hk, n, d) / p.sum(-1, keepdim=True)).transpose(0, 1)
        out.append(o.view(n, hq * d))
        at += n
    return torch.cat(out).to(q.dtype)


def _run_plain(s):
    c = s["case"]
    if c["op"] == "rope":
        x = s["x"].view(c["tokens"], -1, c["d"]).float()
        hq, hk = c["hq"], c["hk"]
        out = [_turned(_norm(u, c["norm"], w), s["pos"], c["rot"], c["pairs"] == "neighbours").flatten(1).to(s["x"].dtype)
               for u, w in ((x[:, :hq], s["wq"]), (x[:, hq:hq + hk], s["wk"]))]
        return tuple(out)
    if c["op"] == "attend":
        return _attend_plain(s, s["x"])
    q = _append_plain(s)
    if c["op"] == "append":
        return (q, *_touched_plain(s))
    return (_attend_plain(s, q), *_touched_plain(s))


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------

def _norm64(x, kind, w):
    x = x.double()
    if kind == "none":
        return x
    mean = x.sum(-1, keepdim=True) / x.shape[-1] if kind == "layer" else torch.zeros_like(x[..., :1])
    var = ((x - mean) ** 2).sum(-1, keepdim=True) / x.shape[-1]
    return (x - mean) * (var + _EPS) ** -0.5 * w.double()


def _turned64(x, pos, rot, neighbours):
    """Each pair as a complex number, times e^(i angle)."""
    freqs = torch.exp(torch.arange(rot // 2, dtype=torch.float64, device=x.device) * (-2.0 / rot * math.log(10000.0)))
    turn = torch.polar(torch.ones_like(freqs), pos.double()[:, None] * freqs)[:, None]
    i = torch.arange(rot // 2, device=x.device)
    a, b = (2 * i, 2 * i + 1) if neighbours else (i, i + rot // 2)
    z = torch.complex(x[..., a], x[..., b]) * turn
    y = x.clone()
    y[..., a], y[..., b] = z.real, z.imag
    return y


def _grid64(v):
    """v rounded to e4m3 by its definition: among all its magnitudes the nearest, found by their midpoints, a tie to
    the even one."""
    mags = [m / 512.0 for m in range(8)] + [(1 + m / 8.0) * 2.0 ** e for e in range(-6, 9) for m in range(8)][:-1]
    grid = torch.tensor(mags, dtype=torch.float64, device=v.device)
    mid = (grid[:-1] + grid[1:]) / 2
    a = v.abs()
    low, high = torch.searchsorted(mid, a), torch.searchsorted(mid, a, right=True)  # they differ at a tie: index - 1 and index
    return grid[torch.where(low % 2 == 0, low, high)] * torch.sign(v)


def _exponent64(top):
    """The least whole e >= -64 with top <= 448 * 2^e (not above 63)."""
    limits = torch.tensor([448.0 * 2.0 ** e for e in range(-64, 63)], dtype=torch.float64, device=top.device)
    return torch.searchsorted(limits, top) - 64


def _two(e):
    powers = torch.tensor([2.0 ** i for i in range(-200, 201)], dtype=torch.float64, device=e.device)
    return powers[e + 200]


def _held64(s, which, i, length):
    """The first `length` tokens of sequence i, token by token: f64 [length, hk, d]."""
    page = s["case"]["page"]
    j = torch.arange(length, device=s["k"].device)
    ids = s["table"][i, j // page].long()
    code = s[which][ids, :, j % page].long()
    mag = torch.where((code & 127) < 8, (code & 7).double() / 512, (8 + (code & 7)).double() * _two((code >> 3 & 15) - 10))
    return mag * (1 - 2 * (code >> 7).double()) * _two(s["scales"][ids, :, "kv".index(which)].long() - 127)[..., None]


def _after64(s, which, new, at, i):
    """The values of sequence i after its rows `new` joined it, block by block."""
    c = s["case"]
    n, length = s["plan"][i]
    page, old = c["page"], length - n
    v = torch.zeros(length, c["hk"], c["d"], dtype=torch.float64, device=new.device)
    if old:
        v[:old] = _held64(s, which, i, old)
    v[old:] = new[at:at + n]
    first = old // page
    for p in range(first, -(-length // page)):
        block = v[p * page:(p + 1) * page]
        fresh = v[max(old, p * page):(p + 1) * page]
        e = _exponent64(fresh.abs().amax(0).amax(-1))
        if p * page < old:
            e = torch.maximum(e, s["scales"][s["table"][i, p].long(), :, "kv".index(which)].long() - 127)
        block.copy_(_grid64(block / _two(e)[:, None]) * _two(e)[:, None])
    return v


def exact(case, seed):
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    c = case
    hq, hk, d = c["hq"], c["hk"], c["d"]
    if c["op"] == "rope":
        x = s["x"].view(c["tokens"], -1, d)
        return tuple(_turned64(_norm64(u, c["norm"], w), s["pos"], c["rot"], c["pairs"] == "neighbours").flatten(1)
                     for u, w in ((x[:, :hq], s["wq"]), (x[:, hq:hq + hk], s["wk"])))
    rows = s["x"].shape[0]
    if c["op"] == "attend":
        q = s["x"].view(rows, hq, d).double()
    else:
        x = s["x"].view(rows, -1, d)
        pos = torch.cat([torch.arange(length - n, length, device=x.device) for n, length in s["plan"]])
        q = _turned64(_norm64(x[:, :hq], c["norm"], s["wq"]), pos, d, False)
        k = _turned64(_norm64(x[:, hq:hq + hk], c["norm"], s["wk"]), pos, d, False)
        v = x[:, hq + hk:].double()
    out, kt, vt, at = [], [], [], 0
    for i, (n, length) in enumerate(s["plan"]):
        if c["op"] == "attend":
            ki, vi = _held64(s, "k", i, length), _held64(s, "v", i, length)
        else:
            ki, vi = _after64(s, "k", k, at, i), _after64(s, "v", v, at, i)
            kt.append(ki[length - s["touched"][i]:].flatten(1))
            vt.append(vi[length - s["touched"][i]:].flatten(1))
        if c["op"] != "append":
            # queries as the layer's attention gets them: of the rows' type
            qi = q[at:at + n].to(s["x"].dtype).double()
            o = torch.empty(n, hq, d, dtype=torch.float64, device=q.device)
            p = torch.arange(length - n, length, device=q.device)
            j = torch.arange(length, device=q.device)
            sees = j[None] <= p[:, None]
            if c["window"]:
                sees &= p[:, None] - j[None] < c["window"]
            for h in range(hq):
                w = torch.softmax((qi[:, h] @ ki[:, h * hk // hq].T / math.sqrt(d)).masked_fill(~sees, -math.inf), -1)
                o[:, h] = w @ vi[:, h * hk // hq]
            out.append(o.flatten(1))
        at += n
    if c["op"] == "attend":
        return torch.cat(out)
    return (q.flatten(1) if c["op"] == "append" else torch.cat(out)), torch.cat(kt), torch.cat(vt)
