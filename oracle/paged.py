"""Rotary positions, the append to a paged 8-bit cache and the attention over it, in float64 from their definitions."""
from __future__ import annotations

import math

import numpy as np

TOP = {"e4m3": 448.0, "int8": 127.0}


def rotate(x, pos, turns, interleaved=False, mscale=1.0, inverse=False):
    """x (T, H, D) float64 rotated by pos (T); turns (rot / 2)."""
    x = np.asarray(x, np.float64)
    turns = np.asarray(turns, np.float64)
    rot = 2 * turns.size
    a = 2.0 * math.pi * np.mod(np.asarray(pos, np.float64)[:, None] * turns, 1.0) * (-1.0 if inverse else 1.0)
    c, s = mscale * np.cos(a)[:, None], mscale * np.sin(a)[:, None]
    ia, ib = (np.arange(0, rot, 2), np.arange(1, rot, 2)) if interleaved else (np.arange(rot // 2),
                                                                              np.arange(rot // 2, rot))
    y = x.copy()
    y[..., ia] = x[..., ia] * c - x[..., ib] * s
    y[..., ib] = x[..., ib] * c + x[..., ia] * s
    return y


def tokens(qsl, lens):
    """(request, position) of each query token of the step; a position is negative where the length is too short."""
    out = []
    for r in range(len(lens)):
        q0, q1 = int(qsl[r]), int(qsl[r + 1])
        out += [(r, int(lens[r]) - q1 + t) for t in range(q0, q1)]
    return out


def smallest_scale(amax, kind):
    if amax == 0:
        return 2.0 ** -126
    e = math.ceil(math.log2(amax / TOP[kind]))
    while 2.0 ** (e - 1) * TOP[kind] >= amax:
        e -= 1
    while 2.0 ** e * TOP[kind] < amax:
        e += 1
    return 2.0 ** max(e, -126)


def half_step(x, scale, kind):
    """How far the nearest code's value may be from x at this scale."""
    x = np.abs(np.asarray(x, np.float64))
    return np.maximum(x * 2.0 ** -4, scale * 2.0 ** -10) if kind == "e4m3" else np.broadcast_to(scale * 0.5, x.shape)


def append(key, value, stored, scales, qsl, lens, bt, kind, slots):
    """What the cache should stand for after the step: (values, scales, tolerance), values (pages, heads, slots, 2 D)
    float64 from `stored` (what it stood for) with the keys and values put in unrounded, and how far a nearest code
    may be from each.  key is already rotated; stored is changed nowhere else."""
    stored, scales = stored.copy(), scales.copy()
    tol = np.zeros_like(stored)
    H, D = key.shape[1:]
    pages = {}
    for t, (r, p) in enumerate(tokens(qsl, lens)):
        if p < 0 or p // slots >= bt.shape[1] or not 0 <= bt[r, p // slots] < stored.shape[0]:
            continue
        pages.setdefault(int(bt[r, p // slots]), []).append((p % slots, t))
    for page, rows in pages.items():
        at = [s for s, _ in rows]
        for h in range(H):
            for i, src in enumerate((key, value)):
                x = src[[t for _, t in rows], h]
                fin = np.abs(x[np.isfinite(x)])
                need = smallest_scale(fin.max() if fin.size else 0.0, kind)
                was = scales[page, h, i]
                now = need if 0 in at else max(was, need)
                cols = slice(i * D, i * D + D)
                if 0 not in at and now > was:
                    tol[page, h, :, cols] = half_step(stored[page, h, :, cols], now, kind)
                if 0 in at:                                # a page started anew: its other slots hold nothing yet
                    tol[page, h, :, cols] = np.inf
                scales[page, h, i] = now
                stored[page, h, at, cols] = x
                tol[page, h, at, cols] = half_step(x, now, kind)
    return stored, scales, tol


def attend(q, kv, qsl, lens, bt, slots, scale, window=0):
    """(o, lse, mass, terms): kv (pages, kv heads, slots, 2 D) float64 values; mass is sum p |v| / sum p, which bounds what
    rounded probabilities do, and terms the largest |q| . |k| scale of each row.  A page outside the cache is NaN."""
    T, Hq, D = q.shape
    Hkv = kv.shape[1]
    o, mass = np.zeros((T, Hq, D)), np.zeros((T, Hq, D))
    lse, terms = np.full((T, Hq), -np.inf), np.zeros((T, Hq))
    for t, (r, p) in enumerate(tokens(qsl, lens)):
        keys = np.arange(max(0, p - window + 1) if window else 0, min(p + 1, bt.shape[1] * slots))
        if not keys.size:
            continue
        pg = bt[r, keys // slots]
        bad = (pg < 0) | (pg >= kv.shape[0])
        rows = kv[np.where(bad, 0, pg), :, keys % slots]
        rows = np.where(bad[:, None, None], np.nan, rows)
        for h in range(Hq):
            k, v = rows[:, h // (Hq // Hkv), :D], rows[:, h // (Hq // Hkv), D:]
            with np.errstate(invalid="ignore"):
                s = k @ q[t, h] * scale
                m = s.max()
                e = np.exp(s - m)
                o[t, h] = e @ v / e.sum()
                mass[t, h] = e @ np.abs(v) / e.sum()
                lse[t, h] = m + np.log(e.sum())
                terms[t, h] = (np.abs(k) @ np.abs(q[t, h]) * abs(scale)).max()
    return o, lse, mass, terms
