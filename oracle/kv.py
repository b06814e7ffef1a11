"""64-bit restatements of the KV-cache operators (rotary positions, append,
attention over a shared prefix and own slots, eviction), straight from their
formulas. numpy only; checkers, never part of the product."""
from __future__ import annotations

import math

import numpy as np


def rope_table(pos, *, rope_dim, theta=1e7, freq_scale=1.0, ext_factor=0.0, attn_factor=1.0, beta_fast=32.0,
               beta_slow=1.0, n_ctx_orig=0, freq_factors=None, **_):
    """Angles [tokens, rope_dim/2] and the magnitude. Float parameters enter as
    the fp32 values that the C struct holds."""
    f = lambda v: float(np.float32(v))
    d, theta, scale = rope_dim, f(theta), f(freq_scale)
    i = np.arange(d // 2, dtype=np.float64)
    freq = theta ** (-2.0 * i / max(d, 1))
    if freq_factors is not None:
        freq = freq / np.asarray(freq_factors, np.float64)
    coef, mag = np.full(d // 2, scale), f(attn_factor)
    if ext_factor != 0.0:
        c = lambda b: d * math.log(n_ctx_orig / (f(b) * 2 * math.pi)) / (2 * math.log(theta))
        lo, hi = max(0, math.floor(c(beta_fast))), min(d - 1, math.ceil(c(beta_slow)))
        r = f(ext_factor) * (1 - np.clip((i - lo) / max(0.001, hi - lo), 0, 1))
        coef = scale * (1 - r) + r
        mag *= 1 + 0.1 * math.log(1 / scale)
    return np.asarray(pos, np.float64)[:, None] * freq * coef, mag


def rope(x, pos, *, layout="half", transpose=False, **kw):
    """x [tokens, heads, D] rotated, in 64 bits."""
    y = np.array(x, np.float64)
    d = kw["rope_dim"]
    a, mag = rope_table(pos, **kw)
    c, s = mag * np.cos(a)[:, None], mag * np.sin(a)[:, None] * (-1 if transpose else 1)
    u, v = (slice(0, d // 2), slice(d // 2, d)) if layout == "half" else (slice(0, d, 2), slice(1, d, 2))
    x1, x2 = y[..., u].copy(), y[..., v].copy()
    y[..., u], y[..., v] = x1 * c - x2 * s, x2 * c + x1 * s
    return y


def attn(q, k, v, lens, k_prefix=None, v_prefix=None, scale=None, weight=None, decay=1.0):
    """q [B, Hq, D], k, v [B, ctx, Hkv, D] -> (o [B, Hq, D], weight or None)."""
    q = np.asarray(q, np.float64)
    b, hq, d = q.shape
    hkv = k.shape[2]
    g = hq // hkv
    scale = d ** -0.5 if scale is None else float(np.float32(scale))
    o = np.zeros((b, hq, d))
    w = None if weight is None else np.array(weight, np.float64)
    dec = float(np.float32(decay))
    for s in range(b):
        n = int(lens[s])
        for j in range(hkv):
            kk, vv = np.asarray(k[s, :n, j], np.float64), np.asarray(v[s, :n, j], np.float64)
            p0 = 0
            if k_prefix is not None:
                p0 = k_prefix.shape[0]
                kk = np.concatenate([np.asarray(k_prefix[:, j], np.float64), kk])
                vv = np.concatenate([np.asarray(v_prefix[:, j], np.float64), vv])
            if kk.shape[0] == 0:
                continue
            sc = q[s, j * g:(j + 1) * g] @ kk.T * scale
            p = np.exp(sc - sc.max(-1, keepdims=True))
            p /= p.sum(-1, keepdims=True)
            o[s, j * g:(j + 1) * g] = p @ vv
            if w is not None and n:
                new = p[:, p0:].sum(0)
                w[s, j, :n] = new if dec == 0.0 else dec * w[s, j, :n] + new
    return o, w


def evict(k, v, weight, slot_pos, lens, pos, budget, n_sink, n_recent):
    """In place on numpy arrays, slot by slot."""
    for s in range(k.shape[0]):
        n = int(lens[s])
        if n <= budget:
            continue
        for j in range(k.shape[2]):
            w, sp = weight[s, j], slot_pos[s, j]
            safe = [bool(sp[t] < n_sink or int(sp[t]) > int(pos[s]) - n_recent) for t in range(n)]
            key = [(math.inf, 1) if safe[t] else (float(w[t]) if w[t] > 0 else 0.0, 0) for t in range(n)]
            order = sorted(range(n), key=lambda t: (-key[t][1], -key[t][0], t))
            kept = set(order[:budget])
            holes = [t for t in range(budget) if t not in kept]
            frm = [t for t in range(budget, n) if t in kept]
            for dst, src in zip(holes, frm):
                for a in (k[s, :, j], v[s, :, j], w, sp):
                    a[dst] = a[src]
        lens[s] = budget
