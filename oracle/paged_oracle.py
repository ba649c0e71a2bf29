"""Plain 64-bit forms of the paged-cache operators, in numpy (test infrastructure).

Written from the operators' definitions: page tables from lengths, rotation of
pairs (the reference's rotary embedding, engine.py:130-158, for any layout),
e4m3 pages with a power-of-two scale per page and head, and causal softmax
attention (engine.py:100-125) of ragged requests.
"""
from __future__ import annotations

import math

import numpy as np


def _e4m3_values():
    """The 127 values 0..448 of e4m3's positive codes 0..126."""
    out = []
    for code in range(127):
        e, m = code >> 3, code & 7
        out.append((m / 8) * 2.0 ** -6 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7))
    return np.array(out)


POSITIVE = _e4m3_values()


def e4m3_encode(x):
    """Bytes of float64 x: nearest value, ties to the even code, saturating; NaN becomes 0."""
    x = np.asarray(x, np.float64)
    a = np.minimum(np.nan_to_num(np.abs(x), nan=0.0, posinf=448.0), 448.0)
    hi = np.clip(np.searchsorted(POSITIVE, a, side="left"), 0, 126)
    lo = np.maximum(hi - 1, 0)
    up, down = POSITIVE[hi] - a, a - POSITIVE[lo]
    code = np.where(up < down, hi, np.where(down < up, lo, np.where(hi % 2 == 0, hi, lo)))
    code = np.where(a == POSITIVE[hi], hi, code)
    return (code + 128 * (np.signbit(x) & ~np.isnan(x))).astype(np.uint8)


def e4m3_decode(b):
    b = np.asarray(b)
    code = b & 127
    v = np.where(code == 127, np.nan, POSITIVE[np.minimum(code, 126)])
    return np.where(b >= 128, -v, v)


def page_scale(top):
    """The smallest 2^e, -40 <= e <= 40, with top <= 448 * 2^e."""
    for e in range(-40, 41):
        if top <= 448 * 2.0 ** e:
            return 2.0 ** e
    return 2.0 ** 40


def plan(starts, q_lens, tables, free, n_free, page, n_rows):
    """(cu_q, kv_lens, positions, slots, tables, n_free), or None where the step does not work out."""
    tables = tables.copy()
    width = tables.shape[1]
    if any(s < 0 or q < 0 or s + q > width * page for s, q in zip(starts, q_lens)) or sum(q_lens) > n_rows:
        return None
    cu, pos, slot = [0], [], []
    for r, (s, q) in enumerate(zip(starts, q_lens)):
        for p in range(s // page, -(-(s + q) // page) if q else 0):
            if tables[r, p] < 0:
                if n_free == 0:
                    return None
                n_free -= 1
                tables[r, p] = free[n_free]
        for x in range(s, s + q):
            pos.append(x)
            slot.append(int(tables[r, x // page]) * page + x % page)
        cu.append(cu[-1] + q)
    pad = n_rows - len(pos)
    return (np.array(cu), np.array(starts) + np.array(q_lens), np.array(pos + [-1] * pad), np.array(slot + [-1] * pad),
            tables, n_free)


def rotate(x, cos, sin, positions, interleaved):
    """x [rows, heads, dim] in float64, rows at position -1 unchanged."""
    out = np.array(x, np.float64)
    half = cos.shape[1]
    for t, pos in enumerate(positions):
        if pos < 0:
            continue
        for i in range(half):
            a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
            c, s = float(cos[pos, i]), float(sin[pos, i])
            u, v = out[t, :, a].copy(), out[t, :, b].copy()
            out[t, :, a], out[t, :, b] = u * c - v * s, u * s + v * c
    return out


def append(pages, scales, x, slots):
    """x [rows, heads, dim] (float64 of the 16-bit values) into copies of pages / scales."""
    pages, scales = pages.copy(), scales.astype(np.float64).copy()
    page = pages.shape[2]
    t = 0
    while t < len(slots):
        if slots[t] < 0:
            t += 1
            continue
        p, lo, n = slots[t] // page, slots[t] % page, 1
        while t + n < len(slots) and slots[t + n] == slots[t] + n and lo + n < page:
            n += 1
        for h in range(pages.shape[1]):
            rows = x[t:t + n, h]
            fine = rows[np.isfinite(rows)]
            need = page_scale(np.abs(fine).max() if fine.size else 0.0)
            old = scales[p, h] if lo else 0.0
            now = max(need, old)
            if lo and need > old:
                pages[p, h, :lo] = e4m3_encode(e4m3_decode(pages[p, h, :lo]) * (old / now))
            scales[p, h] = now
            pages[p, h, lo:lo + n] = e4m3_encode(rows / now)
        t += n
    return pages, scales


def attention(q, k_pages, v_pages, k_scale, v_scale, tables, cu_q, kv_lens, scale=None):
    """(out, lse) in float64; rows without a key give 0 and -inf, padding rows NaN."""
    rows, heads, dim = q.shape
    _, nkv, page, _ = k_pages.shape
    scale = dim ** -0.5 if scale is None else scale
    out = np.full(q.shape, np.nan)
    lse = np.full((rows, heads), np.nan)
    for r in range(len(kv_lens)):
        lo, hi, kv = int(cu_q[r]), int(cu_q[r + 1]), int(kv_lens[r])
        n = -(-kv // page)
        ids = tables[r, :n]
        for h in range(nkv):
            k = (e4m3_decode(k_pages[ids, h]) * k_scale[ids, h][:, None, None]).reshape(-1, dim)[:kv]
            v = (e4m3_decode(v_pages[ids, h]) * v_scale[ids, h][:, None, None]).reshape(-1, dim)[:kv]
            for t in range(lo, hi):
                seen = kv - (hi - 1 - t)
                for g in range(h * (heads // nkv), (h + 1) * (heads // nkv)):
                    if seen <= 0:
                        out[t, g], lse[t, g] = 0.0, -math.inf
                        continue
                    s = scale * (k[:seen] @ q[t, g])
                    top = s.max()
                    e = np.exp(s - top)
                    out[t, g] = e @ v[:seen] / e.sum()
                    lse[t, g] = top + math.log(e.sum())
    return out, lse
