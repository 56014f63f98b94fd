"""Plain 64-bit forms of the low-bit operators (numpy): the 4-bit K/V row
format, attention over given values, the token quantiser and the 8-bit
product.  TEST INFRASTRUCTURE ONLY."""
from __future__ import annotations

import numpy as np


def _bf16_rn(x):
    u = np.asarray(x, np.float32).view(np.uint32)
    return ((u + 0x7FFF + ((u >> 16) & 1)) & np.uint32(0xFFFF0000)).view(np.float32)


def _bf16_up(x):  # x >= 0
    u = np.asarray(x, np.float32).view(np.uint32)
    return ((u + np.uint32(0xFFFF)) & np.uint32(0xFFFF0000)).view(np.float32)


def q4_rows(x):
    """(codes 0..15, s, m) of the rows in x's last dimension; a row that
    cannot be held has s = m = NaN and codes 8."""
    x = np.asarray(x, np.float32)
    bad = ~np.isfinite(x).all(-1)
    d = np.where(bad[..., None], 0, x).astype(np.float64)
    lo, hi = d.min(-1), d.max(-1)
    with np.errstate(over="ignore", invalid="ignore", divide="ignore"):
        m = _bf16_rn(((7 * lo + 8 * hi) / 15).astype(np.float32))
        s = _bf16_up(np.maximum((hi - m.astype(np.float64)) / 7, (m.astype(np.float64) - lo) / 8).astype(np.float32))
        bad |= ~np.isfinite(m) | ~np.isfinite(s)
        near = np.rint((d - m.astype(np.float64)[..., None]) / s.astype(np.float64)[..., None])
    codes = np.where((s > 0)[..., None], np.clip(near, -8, 7), 0) + 8
    codes = np.where(bad[..., None], 8, codes).astype(np.int64)
    return codes, np.where(bad, np.float32(np.nan), s), np.where(bad, np.float32(np.nan), m)


def q4_values(x):
    """The values a 4-bit pool holds for the rows of x (fp32)."""
    c, s, m = q4_rows(x)
    return (m.astype(np.float64)[..., None] + s.astype(np.float64)[..., None] * (c - 8)).astype(np.float32)


def q4_storage(codes, s, m, which, bs):
    """One (block, head) tile's bytes from codes [bs, D] and s, m [bs]."""
    D = codes.shape[1]
    n = codes.reshape(bs, D // 4, 4)
    quads = (n[..., 0] | n[..., 1] << 4 | n[..., 2] << 8 | n[..., 3] << 12).astype(np.uint16)
    if which:  # V: a token pair's quads side by side
        quads = quads.reshape(bs // 2, 2, D // 4).transpose(0, 2, 1)
    params = np.stack([s, m], -1).astype(np.float32).view(np.uint32) >> 16
    return np.concatenate([np.ascontiguousarray(quads).view(np.uint8).ravel(), params.astype(np.uint16).view(np.uint8).ravel()])


def attention64(q, k, v):
    """Causal attention in 64 bits: q [r, Hq, D] the last r of the tokens of
    k, v [n, Hkv, D]."""
    r, hq, d = q.shape
    n, hkv, _ = k.shape
    g = hq // hkv
    out = np.empty((r, hq, d))
    if r == 0:
        return out
    hidden = np.arange(n)[None] > (n - r + np.arange(r))[:, None]
    for h in range(hq):
        with np.errstate(invalid="ignore", over="ignore"):
            x = q[:, h].astype(np.float64) @ k[:, h // g].astype(np.float64).T / np.sqrt(d)
            x = np.where(hidden, -np.inf, x)
            p = np.exp(x - x.max(-1, keepdims=True))
            vv = v[:, h // g].astype(np.float64)
            out[:, h] = np.stack([(p[i, :n - r + i + 1] / p[i].sum()) @ vv[:n - r + i + 1] for i in range(r)])
    return out


def tokens8(x):
    """(codes, fp32 scales) of quantize_tokens."""
    x = np.asarray(x, np.float32)
    bad = ~np.isfinite(x).all(-1)
    d = np.where(bad[:, None], 0, x).astype(np.float64)
    top = np.abs(d).max(-1, initial=0)
    s = np.where(top > 0, (top / 127).astype(np.float32), np.float32(1))
    with np.errstate(divide="ignore", invalid="ignore"):
        c = np.where((s > 0)[:, None], np.clip(np.rint(d / s.astype(np.float64)[:, None]), -127, 127), 0)
    return c.astype(np.int64), np.where(bad, np.float32(np.nan), s)


def product8(codes, s, w, ws):
    """fp32 product of 8-bit rows: exact sums, then one rounding each for the
    sum, the token's and the channel's scale."""
    acc = (codes.astype(np.int64) @ w.astype(np.int64).T).astype(np.float32)
    return acc * np.asarray(s, np.float32)[:, None] * np.asarray(ws, np.float32)[None]
