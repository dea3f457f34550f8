"""Plain restatements in 64 bits (numpy) of the cache's page allocation, of
attention over the cache and of the residual sum with its norms, for the tests."""
from __future__ import annotations

import numpy as np

import kc_mxfp4

I32 = 2 ** 31 - 1


def extend(lens, new, table, stack, count, page, rows):
    """What kv_cache_extend gives, request after request: (lens, count, cu_new,
    cu_seqlens, positions, slots, table)."""
    table = table.copy()
    B, width = table.shape
    free = min(max(int(count), 0), len(stack))
    lens, new = [max(int(x), 0) for x in lens], [max(int(x), 0) for x in new]
    positions, slots = np.full(rows, -1, np.int32), np.full(rows, -1, np.int64)
    asked = used = row = 0
    after, cu_new = [], [0]
    for b in range(B):
        end, total = row + new[b], lens[b] + new[b]
        held = -(-lens[b] // page)
        served = total <= width * page and total <= I32 and end <= rows
        if served:
            ask = -(-total // page) - held
            asked += ask
            served = ask == 0 or asked <= free
            if served:
                for j in range(ask):
                    table[b, held + j] = stack[free - 1 - used - j]
                used += ask
        if served:
            for i in range(new[b]):
                pos = lens[b] + i
                entry = int(table[b, pos // page])
                positions[row + i] = pos
                slots[row + i] = -1 if entry < 0 else entry * page + pos % page
        after.append(total if served else lens[b])
        row = end
        cu_new.append(row)
    cu = np.minimum(np.concatenate([[0], np.cumsum(after, dtype=np.int64)]), I32)
    return (np.array(after, np.int32), np.array([free - used], np.int32), np.minimum(cu_new, I32).astype(np.int32),
            cu.astype(np.int32), positions, slots, table)


def release(finished, lens, table, stack, count, page):
    """What kv_cache_release gives: (lens, count, stack)."""
    stack = stack.copy()
    free = min(max(int(count), 0), len(stack))
    after = []
    for b in range(len(lens)):
        n = max(int(lens[b]), 0)
        if finished[b]:
            for j in range(min(-(-n // page), table.shape[1])):
                if free < len(stack):
                    stack[free] = table[b, j]
                    free += 1
            n = 0
        after.append(n)
    return np.array(after, np.int32), np.array([free], np.int32), stack


def rows_of(pool, fmt):
    """64-bit values [slots, heads, D] of the cache's keys and of its values
    (tensors on any device)."""
    import torch
    out = []
    for codes, scales in (pool[:2], pool[2:]):
        if fmt == "fp8":
            v = codes.view(torch.float8_e4m3fn).double() * scales.double()[..., None]
            out.append(v.flatten(0, 1).cpu().numpy())
        else:
            out.append(kc_mxfp4.values(codes.flatten(0, 1).cpu().numpy(), scales.flatten(0, 1).cpu().numpy()))
    return out


def attention(q, k, v, table, lens, page, scale, window=0):
    """out [B, Hq, D], and what its error goes by: the mean of |v| under the
    weights, and the largest sum of |scale q k|.  k, v [slots, heads, D]."""
    B, Hq, D = q.shape
    H = k.shape[1]
    out, mean, size = np.zeros((B, Hq, D)), np.zeros((B, Hq, D)), np.zeros((B, Hq, 1))
    for b in range(B):
        n = max(int(lens[b]), 0)
        first = max(0, n - window) if window else 0
        if n > table.shape[1] * page:
            out[b] = np.nan
            continue
        pos = np.arange(first, n)
        entry = table[b][pos // page].astype(np.int64)
        if ((entry < 0) | (entry >= k.shape[0] // page)).any():
            out[b] = np.nan
            continue
        if n == 0:
            continue
        at = entry * page + pos % page
        for h in range(Hq):
            kk, vv = k[at, h // (Hq // H)], v[at, h // (Hq // H)]
            s = scale * (kk @ q[b, h])
            p = np.exp(s - s.max())
            p /= p.sum()
            out[b, h], mean[b, h] = p @ vv, p @ np.abs(vv)
            size[b, h] = abs(scale) * (np.abs(kk) @ np.abs(q[b, h])).max()
    return out, mean, size


def attention_tolerance(mean, size, want, D, n, bf16):
    """fp32 scores are off by (D + 12) 2^-23 of the sum of their products' sizes
    (D adds, the scales and the shift by the largest), exp2 by 2^-22, so a
    weight by e = that, and the quotient of two sums by 2 e; n adds of weighted
    values by n 2^-23 each; bf16 queries hold the weights in two bf16 pieces
    (2^-17) and round the output (2^-8).  A weight, or a weight times its row's
    scale, below fp32's smallest normal number 2^-126 may be lost: with the
    largest weight 1, codes up to 448 < 2^9 and scales below 2^8, n 2^-117 2^8."""
    e = 2 * ((D + 12) * 2.0 ** -23 * size + 2.0 ** -21) + (n + 8) * 2.0 ** -23
    lost = n * 2.0 ** -109
    if bf16:
        return (e + 2.0 ** -17) * mean * (1 + 2.0 ** -8) + 2.0 ** -8 * np.abs(want) + lost
    return e * mean + lost


def residual(y, h, gamma, post, gate, alpha, eps):
    """(h', n) and how far fp32 may be off from each: every sum of D squares,
    root, division and product within (D / 2 + 16) 2^-24 of its size."""
    D = y.shape[1]
    e = (D / 2 + 16) * 2.0 ** -24
    b = y if post is None else y / np.sqrt((y * y).mean(-1, keepdims=True) + eps) * post
    add = alpha * b * (1.0 if gate is None else gate)
    x = h + add
    off = e * (np.abs(h) + np.abs(add))
    rms = np.sqrt((x * x).mean(-1, keepdims=True) + eps)
    n = gamma * x / rms
    # the root's own part of h's error: by Cauchy-Schwarz at most its mean square
    off_n = np.abs(gamma) / rms * off + np.abs(n) * (e + np.sqrt((off * off).mean(-1, keepdims=True)) / rms)
    return x, n, off, off_n
