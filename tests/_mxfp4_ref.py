"""Plain float64 / exact-integer restatements of the MXFP4 operators and of the
norms around a residual, written from their definitions (numpy)."""
from __future__ import annotations

import numpy as np
import torch

GRID = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])
DTYPES = {"f32": 0, "f16": 1, "bf16": 2}
EPS = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}  # half a step, relative


def blocks(k):
    return -(-k // 32)


def to_type(x, dtype):
    """float64 array -> (raw host array of `dtype`, the float64 values it holds)."""
    if dtype == "bf16":
        t = torch.from_numpy(np.ascontiguousarray(x, np.float64)).to(torch.bfloat16)
        return t.view(torch.int16).numpy().view(np.uint16), t.double().numpy()
    a = np.asarray(x, np.float64).astype(np.float32 if dtype == "f32" else np.float16)
    return a, a.astype(np.float64)


def from_type(raw, dtype):
    """Raw host bytes of `dtype` -> float64 values."""
    raw = np.ascontiguousarray(raw)
    if dtype == "bf16":
        return torch.from_numpy(raw.view(np.int16).copy()).view(torch.bfloat16).double().numpy()
    return raw.view(np.float32 if dtype == "f32" else np.float16).astype(np.float64)


def np_type(dtype):
    return {"f32": np.float32, "f16": np.float16, "bf16": np.uint16}[dtype]


def quantize(x):
    """x float64 [rows, k] -> (codes [rows, 32 nb] 0..15, scale bytes [rows, nb])."""
    rows, k = x.shape
    nb = blocks(k)
    v = np.zeros((rows, nb * 32))
    v[:, :k] = x
    v = v.reshape(rows, nb, 32)
    bad = ~np.isfinite(v).all(-1)
    amax = np.where(bad, 1.0, np.abs(np.where(np.isfinite(v), v, 0)).max(-1))
    e = np.where(amax > 0, np.frexp(amax)[1] - 3, -127)
    e = np.maximum(e, -127)
    u = np.abs(np.where(np.isfinite(v), v, 0)) * np.ldexp(1.0, -e)[..., None]
    index = np.zeros(u.shape, np.int64)
    for i in range(7):  # the tie between i and i + 1 goes to the even one
        mid = (GRID[i] + GRID[i + 1]) / 2
        index += (u > mid) if i % 2 == 0 else (u >= mid)
    codes = index + 8 * np.signbit(v)
    codes[bad] = 0
    return codes.reshape(rows, -1).astype(np.uint8), np.where(bad, 255, e + 127).astype(np.uint8)


def values(codes, scales, k):
    """Codes [rows, 32 nb], scale bytes [rows, nb] -> float64 [rows, k]."""
    mag = GRID[codes & 7] * np.where(codes & 8, -1.0, 1.0)
    X = np.where(scales == 255, np.nan, np.ldexp(1.0, scales.astype(np.int64) - 127))
    return (mag.reshape(*scales.shape, 32) * X[..., None]).reshape(scales.shape[0], -1)[:, :k]


def pack_codes(codes):
    return (codes[:, 0::2] | (codes[:, 1::2] << 4)).astype(np.uint8)


def unpack_codes(q, rows, k):
    q = q.reshape(rows, blocks(k) * 16)
    out = np.empty((rows, q.shape[1] * 2), np.uint8)
    out[:, 0::2], out[:, 1::2] = q & 15, q >> 4
    return out


def scale_index(rows, k):
    """Byte of every (row, block)'s scale, and the places past the last block: [rows, 4 tiles]."""
    tiles = -(-blocks(k) // 4)
    r, b = np.arange(rows)[:, None], np.arange(4 * tiles)[None]
    return ((r // 128) * tiles + b // 4) * 512 + (r % 32) * 16 + (r % 128) // 32 * 4 + b % 4


def pack_scales(scales, k, fill=0):
    rows, nb = scales.shape
    tiles = -(-nb // 4)
    full = np.zeros((rows, 4 * tiles), np.uint8)
    full[:, :nb] = scales
    out = np.full(-(-rows // 128) * tiles * 512, fill, np.uint8)
    out[scale_index(rows, k)] = full
    return out


def unpack_scales(s, rows, k):
    return s[scale_index(rows, k)][:, :blocks(k)]


def act(v, kind):
    if kind == 1:
        return np.maximum(v, 0)
    if kind == 3:
        with np.errstate(over="ignore"):
            return v / (1 + np.exp(-v))
    return v


def norm(x, kind, w, b, eps):
    if kind == 0:
        return x
    if kind == 2:
        x = x - x.mean(-1, keepdims=True)
    n = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps)
    n = n * w if w is not None else n
    return n + b if b is not None else n
