"""The 4-bit decode block's operators in 64 bits (numpy): MXFP4 blocks, per-head
norm with rotation, attention of a drafted tree over a cache."""
from __future__ import annotations

import numpy as np

LEVELS = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6], np.float64)


def quantize(x: np.ndarray) -> np.ndarray:
    """[rows, cols] floats -> packed bytes [rows, cols / 32 * 17]."""
    rows, cols = x.shape
    b = x.astype(np.float64).reshape(rows, cols // 32, 32)
    top = np.abs(b).max(2)
    e = np.full(top.shape, -127, np.int64)
    ok = np.isfinite(top)
    some = ok & (top > 0)
    e[some] = np.clip(np.floor(np.log2(top[some])).astype(np.int64) - 2, -127, 127)
    a = np.abs(np.where(ok[..., None], b, 0.0)) / np.exp2(e.astype(np.float64))[..., None]
    # the nearest level, a tie to the even code
    d = np.abs(a[..., None] - LEVELS)
    best = d.min(-1, keepdims=True)
    near = d == best
    first, last = near.argmax(-1), 7 - near[..., ::-1].argmax(-1)
    code = np.where(first % 2 == 0, first, last)
    code = np.where(a >= 6, 7, code).astype(np.uint8)
    code |= (np.signbit(b) & ok[..., None]).astype(np.uint8) << 3
    out = np.empty((rows, cols // 32, 17), np.uint8)
    out[..., 0] = np.where(ok, e + 127, 255)
    out[..., 1:] = code[..., :16] | code[..., 16:] << 4
    return out.reshape(rows, -1)


def dequantize(p: np.ndarray) -> np.ndarray:
    """Packed bytes [rows, cols / 32 * 17] -> f64 [rows, cols]."""
    b = p.reshape(p.shape[0], -1, 17)
    code = np.concatenate([b[..., 1:] & 15, b[..., 1:] >> 4], -1)
    v = LEVELS[code & 7] * np.where(code & 8, -1.0, 1.0) * np.exp2(b[..., :1].astype(np.float64) - 127)
    return np.where(b[..., :1] == 255, np.nan, v).reshape(p.shape[0], -1)


def head_norm(x, w, eps):
    """x [..., dh], w [dh]."""
    x = x.astype(np.float64)
    return x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * w.astype(np.float64)


def rotate(x, pos, dims, mode, base):
    """The first dims of x [tokens, heads, dh] turned by pos [tokens]."""
    i = np.arange(dims // 2)
    a = pos.astype(np.float64)[:, None, None] * base ** (-2.0 * i / max(dims, 1))
    u, v = (slice(0, dims, 2), slice(1, dims, 2)) if mode == 0 else (slice(0, dims // 2), slice(dims // 2, dims))
    y = x.copy()
    y[..., u] = x[..., u] * np.cos(a) - x[..., v] * np.sin(a)
    y[..., v] = x[..., u] * np.sin(a) + x[..., v] * np.cos(a)
    return y


def paths(parents) -> np.ndarray:
    """bool [t, t]: token j is i or an ancestor of i; a slot without a token has an empty row."""
    t = len(parents)
    seen = np.zeros((t, t), bool)
    for i in range(t):
        if not -1 <= parents[i] < t:
            continue
        at, steps = i, 0
        while 0 <= at < t and steps <= t:
            if not -1 <= parents[at] < t:
                break
            seen[i, at] = True
            at, steps = parents[at], steps + 1
    return seen


def tree_attn(q, k, vt, parents, past, scale):
    """q [heads, t, dh], k [kv, slots, dh], vt [kv, dh, slots]; -> out, sum p|v| as [t, heads, dh]."""
    heads, t, dh = q.shape
    kv = k.shape[0]
    out, mass = np.zeros((t, heads, dh)), np.zeros((t, heads, dh))
    seen = paths(parents)
    if not 0 <= past <= k.shape[1] - t:
        return out, mass
    for h in range(heads):
        kh, vh = k[h // (heads // kv)].astype(np.float64), vt[h // (heads // kv)].astype(np.float64)
        for i in range(t):
            if not seen[i].any():
                continue
            j = np.concatenate([np.arange(past), past + np.flatnonzero(seen[i])])
            s = kh[j] @ q[h, i].astype(np.float64) * scale
            p = np.exp(s - s.max())
            p /= p.sum()
            out[i, h], mass[i, h] = vh[:, j] @ p, np.abs(vh[:, j]) @ p
    return out, mass
