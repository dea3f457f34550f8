"""Plain restatements in 64 bits (numpy) of the MXFP4 format, of the head norms
with rotation and of the paged cache's addressing, for the tests."""
from __future__ import annotations

import numpy as np

GRID = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=np.float64)
MID = (GRID[1:] + GRID[:-1]) / 2


def encode_e2m1(a: np.ndarray) -> np.ndarray:
    """Codes of values already divided by their scale: nearest, ties to the
    even code, saturated."""
    m = np.abs(a)
    lo = np.searchsorted(MID, m, side="left")    # a tie goes down
    hi = np.searchsorted(MID, m, side="right")   # a tie goes up
    code = np.where(hi % 2 == 0, hi, lo)
    return (code | (np.signbit(a).astype(np.int64) << 3)).astype(np.uint8)


def quantize(x: np.ndarray):
    """(codes [rows, K/2], scales [rows, K/32]) of x [rows, K]."""
    rows, cols = x.shape
    b = np.asarray(x, dtype=np.float64).reshape(rows, cols // 32, 32)
    finite = np.isfinite(b).all(-1)
    b = np.where(finite[..., None], b, 0.0)
    top = np.abs(b).max(-1, initial=0.0)
    e = np.where(top > 0, np.clip(np.frexp(np.where(top > 0, top, 1.0))[1] - 3, -127, 127), 0)
    code = encode_e2m1(np.ldexp(b, -e[..., None]))
    code = np.where(finite[..., None], code, 0).astype(np.uint8).reshape(rows, cols // 2, 2)
    return code[..., 0] | (code[..., 1] << 4), np.where(finite, e + 127, 255).astype(np.uint8)


def values(codes: np.ndarray, scales: np.ndarray) -> np.ndarray:
    """64-bit values of MXFP4 codes [..., K/2] and scales [..., K/32]."""
    c = np.stack([codes & 15, codes >> 4], -1).reshape(*codes.shape[:-1], -1)
    v = np.where(c >= 8, -1.0, 1.0) * GRID[c & 7]
    s = np.where(scales == 255, np.nan, np.ldexp(1.0, scales.astype(np.int64) - 127))
    return v * np.repeat(s, 32, axis=-1)


def norm_rope(x, gamma, cos, sin, pos, eps, interleaved):
    """Heads [T, H, D] in 64 bits, and the size of the two terms of each output."""
    x = np.asarray(x, dtype=np.float64)
    y = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * gamma
    half = cos.shape[1]
    ok = (pos >= 0) & (pos < cos.shape[0])
    c, s = (t.astype(np.float64)[np.where(ok, pos, 0)][:, None, :] if len(t) else np.zeros((len(pos), 1, half))
            for t in (cos, sin))
    ia = np.arange(0, 2 * half, 2) if interleaved else np.arange(half)
    ib = ia + 1 if interleaved else ia + half
    out, size = y.copy(), np.abs(y)
    a, b = y[..., ia], y[..., ib]
    out[..., ia], out[..., ib] = a * c - b * s, b * c + a * s
    size[..., ia], size[..., ib] = np.abs(a * c) + np.abs(b * s), np.abs(b * c) + np.abs(a * s)
    out[pos < 0] = 0.0
    out[pos >= cos.shape[0]] = np.nan
    return out, size


def slots_of(table, cu, page, total):
    """Slot of each token of a packed batch; -1: missing page, -2: no sequence."""
    out = np.full(total, -2, dtype=np.int64)
    for b in range(len(cu) - 1):
        for t in range(max(cu[b], 0), min(cu[b + 1], total)):
            p, off = divmod(t - cu[b], page)
            out[t] = table[b][p] * page + off if p < len(table[b]) and table[b][p] >= 0 else -1
    return out
