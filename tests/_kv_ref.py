"""The paged 8-bit key/value cache, head norms with the rotation and attention, from their definitions in
float64 (contracts in include/dw_cuda.h)."""
import numpy as np

MAGS = np.array([m / 512.0 for m in range(8)] + [(1 + m / 8.0) * 2.0 ** e for e in range(-6, 9) for m in range(8)][:-1])
MID = (MAGS[:-1] + MAGS[1:]) / 2
VALUES = np.concatenate([MAGS, [np.nan], -MAGS, [np.nan]])  # of the 256 codes


def codes(v):
    """The e4m3 codes of v: the nearest magnitude, ties to the even index, 448 at most; NaN 0x7F."""
    a = np.abs(v)
    low, high = np.searchsorted(MID, a), np.searchsorted(MID, a, side="right")
    index = np.where(low % 2 == 0, low, high)
    return np.where(np.isnan(v), 0x7F, index + 128 * np.signbit(v)).astype(np.uint8)


def exponent(top):
    """The least e in -64 .. 63 with top <= 448 * 2^e."""
    return int(np.searchsorted(448.0 * 2.0 ** np.arange(-64, 63), top)) - 64


class Cache:
    def __init__(self, rng, pages, heads, page, d):
        self.page, self.d = page, d
        # whatever an earlier owner left: any codes, NaN among them, any scales of the format
        self.k = rng.integers(0, 256, (pages, heads, page, d), dtype=np.uint8)
        self.v = rng.integers(0, 256, (pages, heads, page, d), dtype=np.uint8)
        self.s = rng.integers(63, 191, (pages, heads, 2), dtype=np.uint8)

    def append(self, pages, old, k, v):
        """k, v float64 [n, heads, d]: the tokens old .. old + n - 1 of the sequence in `pages`."""
        n, heads, _ = k.shape
        bad = ~(np.isfinite(k) & np.isfinite(v)).all(-1)
        for p in range(old // self.page, -(-(old + n) // self.page) if n else 0):
            a, b = max(old, p * self.page), min(old + n, (p + 1) * self.page)
            for h in range(heads):
                good = ~bad[a - old:b - old, h]
                for which, (store, new) in enumerate(((self.k, k), (self.v, v))):
                    x = new[a - old:b - old, h]
                    e = exponent(np.abs(x[good]).max(initial=0.0))
                    block, held = store[pages[p], h], a - p * self.page
                    if held:
                        was = int(self.s[pages[p], h, which]) - 127
                        e = max(e, was)
                        if e != was:
                            block[:held] = codes(VALUES[block[:held]] * 2.0 ** (was - e))
                    c = codes(np.where(good[:, None], x, 0.0) * 2.0 ** -e)
                    c[~good] = 0x7F if which == 0 else 0
                    block[held:held + b - a] = c
                    self.s[pages[p], h, which] = e + 127

    def read(self, which, pages, length):
        store = (self.k, self.v)[which]
        ids = np.asarray(pages[:-(-length // self.page)], np.int64)
        v = VALUES[store[ids]] * 2.0 ** (self.s[ids, :, which].astype(np.float64) - 127)[:, :, None, None]
        return v.transpose(0, 2, 1, 3).reshape(-1, store.shape[1], self.d)[:length]


def norm(x, kind, w, eps):
    if kind == 0:
        return x
    if kind == 2:
        x = x - x.mean(-1, keepdims=True)
    return x / np.sqrt((x * x).mean(-1, keepdims=True) + np.float64(np.float32(eps))) * (1.0 if w is None else w)


def turn(x, positions, freqs, rot, neighbours):
    """x [rows, heads, d]; the first rot values of each head turned."""
    if not rot:
        return x
    t = np.asarray(positions).astype(np.longdouble)[:, None, None] * np.asarray(freqs, np.float64).astype(np.longdouble)
    c, s = np.cos(t).astype(np.float64), np.sin(t).astype(np.float64)
    i = np.arange(rot // 2)
    a, b = (2 * i, 2 * i + 1) if neighbours else (i, i + rot // 2)
    y = x.copy()
    y[..., a], y[..., b] = x[..., a] * c - x[..., b] * s, x[..., a] * s + x[..., b] * c
    return y


def attention(q, k, v, length, scale, causal, window):
    """q [n, hq, d] float64, k, v [length, hk, d]: (out, the mean of |v| under the weights, the largest |t| of
    the logits, the largest sum |q k| scale), each [n, hq, ..]; rows that see nothing give 0."""
    n, hq, d = q.shape
    group = hq // k.shape[1] if length else 1
    out, mean, big, mass = np.zeros((n, hq, d)), np.zeros((n, hq, d)), np.zeros((n, hq, 1)), np.zeros((n, hq, 1))
    for i in range(n):
        p = length - n + i
        hi = min(length, p + 1) if causal else length
        lo = max(0, p + 1 - window) if causal and window else 0
        if hi <= lo:
            continue
        for h in range(hq):
            kk, vv = k[lo:hi, h // group], v[lo:hi, h // group]
            t = (kk @ q[i, h]) * scale
            w = np.exp(t - np.nanmax(t)) if not np.isnan(t).all() else t
            w = w / w.sum()
            out[i, h], mean[i, h] = w @ vv, w @ np.abs(vv)
            big[i, h], mass[i, h] = np.abs(t).max(), (np.abs(kk) @ np.abs(q[i, h])).max() * scale
    return out, mean, big, mass
