"""GPU parity of the KV-cache operators against their 64-bit restatements
(oracle/kv.py), through the Python wrappers on the C ABI.

Tolerances, derived from the roundings:
  rope    the angle enters sincospi as 2t in [-1, 1] rounded to fp32 (2^-25,
          times pi: 9.4e-8 rad), sincospi and the magnitude product round to
          2^-24 each, two products and a sum to 2^-24: at most 2^-21 of
          |x1| + |x2| = at most 2^-20 max|x| m. Then the output's rounding,
          eps/2 of the value (f16: and 2^-25, half its smallest step).
  attn    q enters as two f16 parts, 22 bits; a score's 128 products sum in
          fp32. With S the largest scale * sum|q_i k_i| of a call, a score is
          off by at most 2^-18 S (128 roundings of 2^-24 at worst, and the
          split's), a probability by twice that, the sums of probabilities and
          of p v by 2^-18 at worst: |o - o64| <= (2^-16 S + 2^-17) max|v|. In
          the 2-norm the roundings are independent, sqrt(128) of them in place
          of 128: a tenth of that.
  weight  (2^-16 S + 2^-17) of the weight added, 2^-23 of the old one.
  evict   moves: equal bits.
"""
from __future__ import annotations

import numpy as np
import pytest

from conftest import rng

pytestmark = pytest.mark.gpu
BAD_ARG = 2001


def T(a, dev):
    import torch
    return torch.from_numpy(np.ascontiguousarray(a)).to(dev)


def _torch_dt(name):
    import torch
    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[name]


def _half_step(name):
    return {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}[name]


def _check_rope(got, ref, x, mag, dt, what=""):
    got = got.double().cpu().numpy()
    tol = 2.0 ** -20 * np.abs(x).max() * abs(mag) + _half_step(dt) * np.abs(ref) + (2.0 ** -25 if dt == "f16" else 0)
    bad = np.abs(got - ref) > tol
    assert not bad.any(), f"{what}: {bad.sum()} values, worst {np.abs(got - ref).max():.3e}"


ROPE = [
    dict(head_dim=128, rope_dim=128, layout="interleaved"),
    dict(head_dim=128, rope_dim=64, layout="half"),
    dict(head_dim=80, rope_dim=20, layout="half"),
    dict(head_dim=80, rope_dim=40, layout="interleaved"),
    dict(head_dim=6, rope_dim=2, layout="half", theta=100.0),
    dict(head_dim=2, rope_dim=2, layout="interleaved", theta=100.0),
    dict(head_dim=512, rope_dim=510, layout="interleaved"),
    dict(head_dim=128, rope_dim=0, layout="half"),
    dict(head_dim=128, rope_dim=128, layout="half", theta=1e6, freq_scale=0.25),
    dict(head_dim=128, rope_dim=96, layout="interleaved", theta=1e6, freq_scale=0.125, ext_factor=1.0,
         n_ctx_orig=16384),
    dict(head_dim=256, rope_dim=64, layout="half", theta=1e4, freq_scale=0.5, ext_factor=0.5, attn_factor=0.75,
         n_ctx_orig=4096, beta_fast=16.0, beta_slow=2.0),
]


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("i", range(len(ROPE)))
def test_rope(cuda, dt, i):
    import torch
    from leaninfer_b200 import ops
    from oracle import kv
    kw = dict(theta=1e7) | ROPE[i]
    r = rng(100 + i)
    fac = r.uniform(0.5, 4.0, kw["rope_dim"] // 2).astype(np.float32) if i % 2 else None
    R = ops.Rope(**kw, freq_factors=T(fac, cuda) if fac is not None else None)
    for tokens, heads in ((1, 1), (5, 3), (700, 12)):
        x = T(r.standard_normal((tokens, heads, kw["head_dim"])).astype(np.float32), cuda).to(_torch_dt(dt))
        pos = r.integers(0, 1 << 20, tokens).astype(np.int32)
        pos[0] = [0, -3, 2**31 - 1][tokens % 3]
        ref_kw = dict(kw, freq_factors=fac)
        mag = kv.rope_table(pos, **ref_kw)[1]
        for tr in (False, True):
            ref = kv.rope(x.double().cpu().numpy(), pos, transpose=tr, **ref_kw)
            _check_rope(ops.rope(R, x, T(pos, cuda), transpose=tr), ref, x.double().cpu().numpy(), mag, dt,
                        f"{tokens}x{heads} transpose={tr}")
    assert ops.device_status() == 0


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("offset,gap", [(0, 0), (1, 3), (2, 2), (4, 8), (8, 4)])
def test_rope_strides_alignment_and_in_place(cuda, dt, offset, gap):
    """A slice of a wider, possibly misaligned projection, head-major too, and
    in place: the values around the slice stay."""
    import torch
    from leaninfer_b200 import ops
    from oracle import kv
    r = rng(200 + offset)
    kw = dict(head_dim=64, rope_dim=32, layout="half", theta=1e5)
    R = ops.Rope(**kw)
    tokens, heads = 37, 5
    base = T(r.standard_normal(offset + tokens * (heads * 64 + gap)).astype(np.float32), cuda).to(_torch_dt(dt))
    wide = base[offset:].view(tokens, heads * 64 + gap)
    x = wide[:, :heads * 64].view(tokens, heads, 64)
    pos = r.integers(0, 9999, tokens).astype(np.int32)
    x64 = x.double().cpu().numpy()
    ref = kv.rope(x64, pos, **kw)
    _check_rope(ops.rope(R, x, T(pos, cuda)), ref, x64, 1.0, dt, "out of place")
    hm = x.transpose(0, 1).contiguous().transpose(0, 1)                      # head-major storage
    _check_rope(ops.rope(R, hm, T(pos, cuda)), ref, x64, 1.0, dt, "head-major")
    before = base.clone()
    ops.rope(R, x, T(pos, cuda), out=x)
    _check_rope(x, ref, x64, 1.0, dt, "in place")
    around = torch.ones_like(base, dtype=torch.bool)
    around[offset:].view(tokens, -1)[:, :heads * 64] = False
    assert torch.equal(base[around], before[around])


def test_rope_transpose_is_the_gradient(cuda):
    """<dy, R x> differentiated by x: against the transposed call, and against
    central differences of the fp32 forward (a linear map: the difference
    quotient is exact up to the forward's rounding, 2^-20 * 2 / step)."""
    import torch
    from leaninfer_b200 import ops
    r = rng(300)
    R = ops.Rope(head_dim=32, rope_dim=16, layout="interleaved", theta=1e4, attn_factor=1.25)
    x, dy = (T(r.standard_normal((3, 2, 32)).astype(np.float32), cuda) for _ in range(2))
    pos = T(np.array([0, 7, 12345], np.int32), cuda)
    grad = ops.rope(R, dy, pos, transpose=True)
    for _ in range(20):
        t, h, d = int(r.integers(3)), int(r.integers(2)), int(r.integers(32))
        e = torch.zeros_like(x)
        e[t, h, d] = 0.5
        num = ((ops.rope(R, x + e, pos).double() - ops.rope(R, x - e, pos).double()) * dy.double()).sum()
        scale = float(x.abs().max() * 1.25 * dy.abs().sum())
        assert abs(float(num) - float(grad[t, h, d])) <= 2.0 ** -19 * scale


def test_rope_moves_cached_keys(cuda):
    """Keys rotated to position p, then by d on the fp16 cache rows, are the
    keys rotated to p + d (two f16 roundings)."""
    import torch
    from leaninfer_b200 import ops
    from oracle import kv
    r = rng(310)
    kw = dict(head_dim=128, rope_dim=64, layout="half", theta=1e6)
    R = ops.Rope(**kw)
    x = r.standard_normal((50, 4, 128)).astype(np.float32)
    pos, d = r.integers(0, 30000, 50).astype(np.int32), r.integers(-20000, 20000, 50).astype(np.int32)
    rows = ops.rope(R, T(x, cuda), T(pos, cuda)).half()
    ops.rope(R, rows, T(d, cuda), out=rows)
    ref = kv.rope(x, pos.astype(np.int64) + d, **kw)
    got = rows.double().cpu().numpy()
    assert np.abs(got - ref).max() <= 3 * 2.0 ** -11 * np.abs(x).max() * np.sqrt(2)


# --------------------------------------------------------------------------
def _cache(r, dev, B, ctx, Hkv, lens, P=0, weight=True, stale=float("nan")):
    """numpy arrays of a cache and the KVCache over their device copies; slots
    past a length hold `stale` (and infinities)."""
    from leaninfer_b200 import ops
    f16 = lambda *s: r.standard_normal(s).astype(np.float16)
    c = dict(k=f16(B, ctx, Hkv, 128), v=f16(B, ctx, Hkv, 128), lens=np.asarray(lens, np.int32),
             kp=f16(P, Hkv, 128) if P else None, vp=f16(P, Hkv, 128) if P else None,
             weight=r.random((B, Hkv, ctx)).astype(np.float32) if weight else None,
             slot_pos=np.broadcast_to(np.arange(ctx, dtype=np.int32), (B, Hkv, ctx)).copy())
    if stale is not None:
        for s, n in enumerate(c["lens"]):
            if 0 <= n <= ctx:
                c["k"][s, n:], c["v"][s, n:] = stale, stale
                c["v"][s, n::2] = np.inf
    t = {k: T(v, dev) if v is not None else None for k, v in c.items()}
    return c, t, ops.KVCache(t["k"], t["v"], t["lens"], k_prefix=t["kp"], v_prefix=t["vp"], weight=t["weight"],
                             slot_pos=t["slot_pos"])


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("layout,rope_dim", [("half", 64), ("interleaved", 128), ("none", 0)])
@pytest.mark.parametrize("mode", ["step", "prompt"])
def test_append(cuda, dt, layout, rope_dim, mode):
    import torch
    from leaninfer_b200 import ops
    from oracle import kv
    r = rng(400 + rope_dim)
    B, ctx, Hkv, G = 5, 40, 3, 4
    lens = np.array([1, 40, 17, 9, 30], np.int32)
    c, t, cache = _cache(r, cuda, B, ctx, Hkv, lens)
    kw = dict(head_dim=128, rope_dim=rope_dim, layout=layout, theta=1e6)
    R = ops.Rope(**kw) if layout != "none" else None
    if mode == "step":
        seq, slot, args = np.arange(B), lens - 1, {}
    else:
        seq, slot = np.concatenate([np.full(7, s) for s in (3, 0, 4)]), np.concatenate([np.arange(a, a + 7) for a in
                                                                                       (0, 33, 11)])
        args = dict(seq=T(seq.astype(np.int32), cuda), slot=T(slot.astype(np.int32), cuda))
    n = len(seq)
    pos = r.integers(0, 50000, n).astype(np.int32)
    proj = T(r.standard_normal((n, (G + 2) * Hkv * 128 + 12)).astype(np.float32), cuda).to(_torch_dt(dt))
    cut = lambda a, b: proj[:, a * 128:b * 128].view(n, b - a, 128)
    q, k, v = cut(0, G * Hkv), cut(G * Hkv, (G + 1) * Hkv), cut((G + 1) * Hkv, (G + 2) * Hkv)
    q64, k64, v64 = (a.double().cpu().numpy() for a in (q, k, v))
    got_q = cache.append(k, v, T(pos, cuda), q=q, rope=R, **args)
    if R is not None:
        q_ref, k_ref = kv.rope(q64, pos, **kw), kv.rope(k64, pos, **kw)
    else:
        q_ref, k_ref = q64, k64
    _check_rope(got_q, q_ref, q64, 1.0, dt, "q")
    kc, vc = t["k"].cpu().numpy(), t["v"].cpu().numpy()
    tol = 2.0 ** -20 * np.abs(k64).max() + 2.0 ** -25
    assert np.all(np.abs(kc[seq, slot].astype(np.float64) - k_ref) <= tol + 2.0 ** -11 * np.abs(k_ref))
    assert np.all(np.abs(vc[seq, slot].astype(np.float64) - v64) <= 2.0 ** -11 * np.abs(v64) + 2.0 ** -25)
    w, sp = t["weight"].cpu().numpy(), t["slot_pos"].cpu().numpy()
    assert np.all(w[seq, :, slot] == 0) and np.all(sp[seq, :, slot] == pos[:, None])
    rest = np.ones((B, ctx), bool)
    rest[seq, slot] = False
    bits = lambda a: a.view(np.uint16)
    assert np.array_equal(bits(kc)[rest], bits(c["k"])[rest]) and np.array_equal(bits(vc)[rest], bits(c["v"])[rest])
    rest_h = np.broadcast_to(rest[:, None], w.shape)
    assert np.array_equal(w[rest_h], c["weight"][rest_h]) and np.array_equal(sp[rest_h], c["slot_pos"][rest_h])
    assert np.array_equal(t["lens"].cpu().numpy(), lens) and ops.device_status() == 0
    # in place, and without queries: the same cache rows
    before = t["k"].clone()
    assert cache.append(k, v, T(pos, cuda), rope=R, **args) is None
    cache.append(k, v, T(pos, cuda), q=q, q_out=q, rope=R, **args)
    assert torch.equal(q, got_q) and torch.equal(t["k"].view(torch.int16), before.view(torch.int16))


def test_append_outside_the_cache(cuda):
    """Sequences and slots outside write nothing and raise the device flag;
    the other tokens are written and every q is rotated."""
    import torch
    from leaninfer_b200 import ops
    r = rng(450)
    c, t, cache = _cache(r, cuda, 3, 8, 2, [0, 9, 4])
    n = 6
    q, k, v = (T(r.standard_normal((n, h, 128)).astype(np.float32), cuda) for h in (4, 2, 2))
    pos = T(np.arange(n, dtype=np.int32), cuda)
    seq, slot = T(np.array([0, 1, -1, 3, 2, 2], np.int32), cuda), T(np.array([-1, 8, 0, 0, 7, 0], np.int32), cuda)
    R = ops.Rope(head_dim=128, rope_dim=64)
    out = cache.append(k, v, pos, q=q, rope=R, seq=seq, slot=slot)
    assert ops.device_status() == BAD_ARG
    assert torch.equal(out, ops.rope(R, q, pos))
    kc, c16 = t["k"].cpu().numpy().view(np.uint16), c["k"].view(np.uint16)
    same = np.array([[np.array_equal(kc[s, i], c16[s, i]) for i in range(8)] for s in range(3)])
    assert not same[2, 7] and not same[2, 0] and same.sum() == 22
    # lengths 0 and 9 of 8 slots have no last slot
    cache.append(k[:3], v[:3], pos[:3], rope=R)
    assert ops.device_status() == BAD_ARG and ops.device_status() == 0
    kc2 = t["k"].cpu().numpy().view(np.uint16)
    assert np.array_equal(kc2[:2], kc[:2]) and not np.array_equal(kc2[2, 3], kc[2, 3])


# --------------------------------------------------------------------------
def _attn_check(cuda, r, B, P, ctx, lens, Hkv, G, *, weight=True, decay=1.0, q_scale=1.5, k_scale=1.0, gap=0, scale=None,
                graph=False):
    import torch
    from leaninfer_b200 import ops
    from oracle import kv
    c, t, cache = _cache(r, cuda, B, ctx, Hkv, lens, P, weight)
    if k_scale != 1.0:
        for name in ("k", "kp"):
            if c[name] is not None:
                c[name] = (c[name].astype(np.float32) * k_scale).astype(np.float16)
                t[name].copy_(T(c[name], cuda))
    wide = (q_scale * r.standard_normal((B, Hkv * G * 128 + gap))).astype(np.float32)
    q = wide[:, :Hkv * G * 128].reshape(B, Hkv * G, 128)
    qd = T(wide, cuda)[:, :Hkv * G * 128].view(B, Hkv * G, 128)
    if graph:
        out = torch.full((B, Hkv * G, 128), 7.0, device=cuda)
        w0 = t["weight"].clone() if weight else None
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            cache.decode(qd, decay=decay, out=out, scale=scale)           # warm-up off the capture
        s.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            cache.decode(qd, decay=decay, out=out, scale=scale)
        out.fill_(3.0)
        if weight:
            t["weight"].copy_(w0)
        g.replay()
        got = out
    else:
        got = cache.decode(qd, decay=decay, scale=scale)
    sane = np.where((c["lens"] < 0) | (c["lens"] > ctx), 0, c["lens"])
    ref, w_ref = kv.attn(q, c["k"], c["v"], sane, c["kp"], c["vp"], weight=c["weight"], decay=decay, scale=scale)
    got = got.double().cpu().numpy()
    sc = 128 ** -0.5 if scale is None else scale
    kmax = 0.0
    for s in range(B):
        for k in (c["k"][s, :sane[s]], c["kp"]):
            if k is not None and k.size:
                kk = np.abs(k.astype(np.float64))
                kmax = max(kmax, float(np.einsum("hgd,thd->hgt", np.abs(q[s].astype(np.float64)).reshape(Hkv, G, 128),
                                                 kk).max()))
    S = abs(sc) * kmax
    vmax = max([np.abs(c["v"][s, :sane[s]].astype(np.float64)).max(initial=0) for s in range(B)] +
               [np.abs(c["vp"].astype(np.float64)).max() if P else 0.0])
    tol = 2.0 ** -16 * S + 2.0 ** -17
    assert np.isfinite(got).all()
    worst = np.abs(got - ref).max(initial=0)
    assert worst <= tol * vmax, f"worst {worst:.3e}, allowed {tol * vmax:.3e}"
    norm = np.linalg.norm(ref)
    assert np.linalg.norm(got - ref) <= 0.1 * tol * max(norm, 1e-30), (np.linalg.norm(got - ref) / norm, 0.1 * tol)
    if weight:
        w = t["weight"].double().cpu().numpy()
        for s in range(B):
            n = sane[s]
            assert np.array_equal(w[s, :, n:], c["weight"][s, :, n:].astype(np.float64))    # past the length: untouched
            old = 0.0 if decay == 0.0 else np.abs(decay * c["weight"][s, :, :n])
            new = np.abs(w_ref[s, :, :n] - (0.0 if decay == 0.0 else float(np.float32(decay)) *
                                            c["weight"][s, :, :n].astype(np.float64)))
            assert np.all(np.abs(w[s, :, :n] - w_ref[s, :, :n]) <= tol * new + 2.0 ** -22 * (old + new) + 1e-37)
    kc = t["k"].cpu().numpy()
    assert np.array_equal(kc.view(np.uint16), c["k"].view(np.uint16))
    assert ops.device_status() == (BAD_ARG if (sane != c["lens"]).any() else 0)


ATTN = [
    # B, P, ctx, lens, Hkv, G
    (1, 0, 1, [1], 1, 1),
    (1, 1, 4, [0], 1, 5),
    (2, 0, 5, [0, 5], 2, 4),                         # a row without tokens
    (3, 129, 300, [0, 128, 300], 2, 5),
    (4, 128, 16, [16, 15, 1, 0], 1, 8),
    (1, 1000, 130, [129], 8, 5),
    (5, 63, 70, [1, 64, 65, 33, 17], 3, 3),
    (6, 257, 90, [90, 2, 31, 32, 16, 0], 2, 7),
    (9, 300, 50, list(range(9)), 1, 16),             # 144 rows: two row tiles
    (3, 40, 33, [33, 8, 20], 2, 13),
    (26, 513, 20, [20] * 26, 1, 5),                  # 130 rows, the second tile nearly empty
    (70, 300, 40, [i % 41 for i in range(70)], 1, 5),        # 350 rows: three row tiles
    (130, 200, 9, [i % 10 for i in range(130)], 2, 4),       # 520 rows: five
    (2, 9000, 3000, [3000, 1], 1, 2),
    (40, 0, 700, [700 - 17 * i for i in range(40)], 2, 6),
    (300, 5, 3, [i % 4 for i in range(300)], 1, 1),
]


@pytest.mark.parametrize("case", range(len(ATTN)))
def test_attention(cuda, case):
    B, P, ctx, lens, Hkv, G = ATTN[case]
    _attn_check(cuda, rng(500 + case), B, P, ctx, lens, Hkv, G, decay=[1.0, 0.0, 0.75][case % 3])


@pytest.mark.parametrize("kw", [
    dict(weight=False), dict(gap=20), dict(q_scale=1e6, scale=1e-7), dict(q_scale=1e-20), dict(q_scale=0.0),
    dict(q_scale=40.0), dict(k_scale=1000.0, scale=1e-4), dict(scale=0.0), dict(scale=-0.3), dict(graph=True),
    dict(graph=True, weight=False)])
def test_attention_variants(cuda, kw):
    """No weights, strided q, q beyond the f16 range, tiny, zero and sharp
    queries, keys near the f16 range's end, other scales, a captured graph."""
    _attn_check(cuda, rng(600), 7, 333, 200, [200, 0, 1, 64, 100, 199, 16], 2, 5, **kw)


# Prefixes beyond the size that goes with the own tokens (30 MB, read once per
# sequence): the tensor-core kernel.
PREFIX = [
    # B, P, ctx, lens, Hkv, G
    (2, 40000, 40, [40, 7], 1, 8),                            # 16 rows: one row tile, alternate token tiles
    (9, 8200, 50, list(range(9)), 1, 16),                     # 144 rows: two row tiles
    (26, 2500, 20, [20] * 26, 1, 5),                          # 130 rows, the second tile nearly empty
    (70, 1000, 40, [i % 41 for i in range(70)], 1, 5),        # 350 rows: three row tiles
    (70, 7001, 9, [i % 10 for i in range(70)], 2, 5),         # three, in a pair and a single
    (130, 300, 9, [i % 10 for i in range(130)], 2, 4),        # 520 rows: five
    (620, 100, 3, [i % 4 for i in range(620)], 1, 1),         # five row tiles of one token tile each
    (300, 128, 40, [i % 41 for i in range(300)], 2, 3),       # one whole token tile
    (40, 769, 1, [i % 2 for i in range(40)], 2, 7),
    (64, 4096, 2, [0] * 64, 1, 6),                            # no own tokens
]


@pytest.mark.parametrize("case", range(len(PREFIX)))
def test_attention_over_a_large_prefix(cuda, case):
    B, P, ctx, lens, Hkv, G = PREFIX[case]
    assert B > 1 and B * Hkv * P * 512 > 30 << 20
    _attn_check(cuda, rng(560 + case), B, P, ctx, lens, Hkv, G, decay=[1.0, 0.0, 0.75][case % 3])


@pytest.mark.parametrize("kw", [
    dict(weight=False), dict(gap=20), dict(q_scale=1e6, scale=1e-7), dict(q_scale=1e-20), dict(q_scale=0.0),
    dict(q_scale=40.0), dict(k_scale=1000.0, scale=1e-4), dict(scale=0.0), dict(scale=-0.3), dict(graph=True),
    dict(graph=True, weight=False)])
def test_large_prefix_variants(cuda, kw):
    """The variants above on the tensor-core kernel."""
    _attn_check(cuda, rng(600), 20, 1700, 70, [(i * 13) % 71 for i in range(20)], 2, 5, **kw)


# On both sides of 296 rows the join takes its rows differently: one a warp, four a warp.
ROWS = [
    # B, P, ctx, lens, Hkv, G
    (5, 9910, 3, [0, 1, 2, 2, 0], 1, 16),                     # few rows, hundreds of pieces each
    (1, 20011, 9, [4], 1, 1),
    (27, 6001, 300, [i * 11 for i in range(27)], 2, 3),
    (37, 1700, 64, [i + 7 for i in range(37)], 1, 8),         # 296 rows
    (99, 1000, 20, [i % 21 for i in range(99)], 1, 3),        # 297
    (201, 123, 1, [i % 2 for i in range(201)], 4, 2),         # a prefix of one token tile, four row tiles
    (60, 0, 1500, [1500 - 25 * i for i in range(60)], 1, 8),  # four rows a warp, many pieces each
]


@pytest.mark.parametrize("case", range(len(ROWS)))
def test_attention_joins_few_and_many_rows(cuda, case):
    B, P, ctx, lens, Hkv, G = ROWS[case]
    _attn_check(cuda, rng(620 + case), B, P, ctx, lens, Hkv, G, decay=[1.0, 0.0, 0.75][case % 3])


@pytest.mark.parametrize("kw", [
    dict(weight=False), dict(gap=20), dict(q_scale=0.0), dict(scale=0.0), dict(scale=-0.3), dict(graph=True),
    dict(graph=True, weight=False)])
@pytest.mark.parametrize("P", [0, 900])
def test_many_rows_variants(cuda, P, kw):
    """The variants above with 440 rows."""
    _attn_check(cuda, rng(640), 88, P, 70, [(i * 13) % 71 for i in range(88)], 1, 5, **kw)


def test_large_prefix_growing_scores(cuda):
    """Scores that rise along the prefix by far more than the lag of the
    running maximum, and fall, and jump: every rescaling path."""
    import torch
    from leaninfer_b200 import ops
    from oracle import kv
    r = rng(630)
    B, P, Hkv, G = 24, 3000, 1, 4
    c, t, cache = _cache(r, cuda, B, 8, Hkv, [8] * B, P, weight=False)
    ramp = np.concatenate([np.linspace(-3, 3, 1500), np.linspace(3, -3, 1200), np.full(299, -2.0), [6.0]])
    c["kp"] = (0.05 * c["kp"].astype(np.float32) + ramp[:, None, None]).astype(np.float16)
    t["kp"].copy_(T(c["kp"], cuda))
    q = (r.standard_normal((B, G, 128)) * 0.2 + r.choice([-0.3, 0.3, 0.05], (B, G, 1))).astype(np.float32)
    got = cache.decode(T(q, cuda)).double().cpu().numpy()
    ref, _ = kv.attn(q, c["k"], c["v"], c["lens"], c["kp"], c["vp"])
    S = float(np.abs(q).astype(np.float64).sum(-1).max() * np.abs(c["kp"].astype(np.float64)).max()) * 128 ** -0.5
    assert np.abs(got - ref).max() <= (2.0 ** -16 * S + 2.0 ** -17) * 5
    assert ops.device_status() == 0


def test_attention_bad_lengths(cuda):
    """Lengths outside the cache count as no own slots and raise the flag."""
    _attn_check(cuda, rng(610), 4, 70, 20, [21, -1, 20, 2**31 - 1], 2, 3)
    _attn_check(cuda, rng(611), 20, 1700, 20, [21, -1, 20, 2**31 - 1] * 5, 2, 3)


def test_empty_calls(cuda):
    """No tokens, no sequences: nothing happens."""
    import torch
    from leaninfer_b200 import ops
    R = ops.Rope(head_dim=128, rope_dim=64)
    none = torch.empty(0, device=cuda, dtype=torch.int32)
    assert ops.rope(R, torch.empty(0, 3, 128, device=cuda), none).shape == (0, 3, 128)
    k = torch.zeros(2, 4, 2, 128, device=cuda, dtype=torch.float16)
    cache = ops.KVCache(k, k.clone(), torch.ones(2, device=cuda, dtype=torch.int32))
    z = torch.empty(0, 2, 128, device=cuda)
    assert cache.append(z, z, none) is None and cache.append(z, z, none, q=z).shape == (0, 2, 128)
    k0 = k[:0]
    cache = ops.KVCache(k0, k0.clone(), none, weight=torch.empty(0, 2, 4, device=cuda),
                        slot_pos=torch.empty(0, 2, 4, device=cuda, dtype=torch.int32))
    assert cache.decode(torch.empty(0, 4, 128, device=cuda)).shape == (0, 4, 128)
    cache.evict(none, 2)
    assert ops.device_status() == 0


def test_output_over_the_queries(cuda):
    """decode with out = q, and many sequences (more than the length scan's
    entries) of very different lengths."""
    from leaninfer_b200 import ops
    from oracle import kv
    r = rng(640)
    B, ctx = 4500, 5
    lens = r.integers(0, ctx + 1, B).astype(np.int32)
    lens[1000:3500] = 0
    c, t, cache = _cache(r, cuda, B, ctx, 1, lens, 0, weight=True)
    q = r.standard_normal((B, 2, 128)).astype(np.float32)
    qd = T(q, cuda)
    assert cache.decode(qd, out=qd) is qd
    ref, w_ref = kv.attn(q, c["k"], c["v"], lens, weight=c["weight"])
    assert np.linalg.norm(qd.double().cpu().numpy() - ref) <= 1e-5 * np.linalg.norm(ref)
    assert np.abs(t["weight"].double().cpu().numpy() - w_ref).max() <= 1e-5
    assert ops.device_status() == 0


def test_attention_is_deterministic_and_stream_ordered(cuda):
    """Two caches decoded in turn on two streams, twice: the same bits."""
    import torch
    r = rng(620)
    sets = []
    for P in (2000, 100):
        c, t, cache = _cache(r, cuda, 20, 500, 2, list(range(0, 500, 25)), P)
        q = T(r.standard_normal((20, 10, 128)).astype(np.float32), cuda)
        sets.append((cache, q, cache.decode(q, decay=0.0), t["weight"]))
    torch.cuda.synchronize()
    first = [(o.clone(), w.clone()) for _, _, o, w in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    again = []
    for _ in range(3):
        for (cache, q, _, _), s in zip(sets, streams):
            with torch.cuda.stream(s):
                again.append(cache.decode(q, decay=0.0))
    torch.cuda.synchronize()
    for i, o in enumerate(again):
        assert torch.equal(o, first[i % 2][0])
    for (_, _, _, w), (_, w0) in zip(sets, first):
        assert torch.equal(w, w0)


# --------------------------------------------------------------------------
def _evict_check(cuda, r, B, ctx, Hkv, lens, budget, n_sink, n_recent, weights, shuffle=True):
    import torch
    from leaninfer_b200 import ops
    from oracle import kv
    c, t, cache = _cache(r, cuda, B, ctx, Hkv, lens, stale=7.0)
    c["weight"] = weights((B, Hkv, ctx)).astype(np.float32)
    if shuffle:
        for s in range(B):
            n = max(0, min(int(lens[s]), ctx))
            for j in range(Hkv):
                c["slot_pos"][s, j, :n] = r.permutation(n)
    t["weight"].copy_(T(c["weight"], cuda))
    t["slot_pos"].copy_(T(c["slot_pos"], cuda))
    pos = np.maximum(c["lens"] - 1, 0).astype(np.int32)
    cache.evict(T(pos, cuda), budget, n_sink=n_sink, n_recent=n_recent)
    torch.cuda.synchronize()
    bad = (c["lens"] < 0) | (c["lens"] > ctx)
    ref_len = np.where(bad, 0, c["lens"])
    kv.evict(c["k"], c["v"], c["weight"], c["slot_pos"], ref_len, pos, budget, n_sink, n_recent)
    assert np.array_equal(t["lens"].cpu().numpy(), np.where(bad, c["lens"], ref_len))
    assert np.array_equal(t["slot_pos"].cpu().numpy(), c["slot_pos"])
    assert np.array_equal(t["weight"].cpu().numpy().view(np.uint32), c["weight"].view(np.uint32))
    for a, b in ((t["k"], c["k"]), (t["v"], c["v"])):
        assert np.array_equal(a.cpu().numpy().view(np.uint16), b.view(np.uint16))
    assert ops.device_status() == (BAD_ARG if bad.any() else 0)


EVICT = [
    # B, ctx, Hkv, lens, budget, sink, recent
    (1, 1, 1, [1], 0, 0, 0),
    (1, 2, 1, [2], 1, 0, 0),
    (1, 2, 1, [2], 1, 1, 0),
    (2, 40, 3, [40, 33], 32, 4, 8),
    (4, 100, 2, [100, 0, 64, 65], 64, 0, 64),
    (3, 1000, 2, [1000, 999, 501], 500, 4, 100),
    (3, 1000, 2, [1000, 1000, 10], 0, 0, 0),
    (2, 4097, 1, [4097, 4096], 4096, 4, 256),
    (2, 3000, 2, [3000, 2900], 31, 1, 30),
    (2, 300, 2, [300, 200], 300, 0, 0),
    (1, 60000, 1, [59999], 30011, 4, 1000),             # more slots than the keys' shared memory holds
    (1, 49152, 1, [49152], 40000, 4, 100),              # as many as it holds
    (1, 9000, 2, [9000], 3000, 4, 2900),                # more moves than the selecting block makes itself
    (5, 37, 2, [37, 38, -1, 36, 2**31 - 1], 20, 2, 3),  # lengths outside the cache
]


@pytest.mark.parametrize("case", range(len(EVICT)))
def test_evict(cuda, case):
    r = rng(700 + case)
    _evict_check(cuda, r, *EVICT[case], weights=lambda s: r.random(s) ** 6)


@pytest.mark.parametrize("kind", ["equal", "zero", "few", "special", "nearby", "descending"])
def test_evict_weights(cuda, kind):
    """Ties everywhere, a handful of values, NaN, infinities, negative and
    subnormal weights, weights that differ in the last bits, everything kept
    in the front or at the back."""
    r = rng(750)

    def weights(shape):
        if kind == "equal":
            return np.full(shape, 0.25)
        if kind == "zero":
            return np.zeros(shape)
        if kind == "few":
            return r.integers(0, 3, shape)
        if kind == "special":
            return r.choice(np.array([np.nan, np.inf, -np.inf, -1.0, -0.0, 0.0, 1e-42, 1.0, 3e38], np.float32), shape)
        if kind == "nearby":
            return (np.float32(1.0).view(np.uint32) + r.integers(0, 9, shape).astype(np.uint32)).view(np.float32)
        return np.broadcast_to(-np.arange(shape[-1]) + 2000.0, shape)

    _evict_check(cuda, r, 3, 777, 2, [777, 700, 400], 399, 3, 50, weights, shuffle=kind != "descending")


@pytest.mark.parametrize("budget,pos_of", [(0, -1), (0, 10**9), (16, -1), (16, 2**31 - 1), (16, -2**31), (40, 10**9)])
def test_evict_positions_that_protect_everything(cuda, budget, pos_of):
    """Positions that no token has (a table that was never filled): all slots
    protected, so ties go to the lowest; a budget of 0 keeps none even so."""
    import torch
    from leaninfer_b200 import ops
    from oracle import kv
    r = rng(760)
    c, t, cache = _cache(r, cuda, 2, 50, 2, [50, 30], stale=7.0)
    c["slot_pos"][:] = pos_of
    t["slot_pos"].fill_(pos_of)
    pos = np.array([49, 29], np.int32)
    cache.evict(T(pos, cuda), budget, n_sink=0, n_recent=0)
    lens = c["lens"].copy()
    kv.evict(c["k"], c["v"], c["weight"], c["slot_pos"], lens, pos, budget, 0, 0)
    assert np.array_equal(t["lens"].cpu().numpy(), lens)
    for a, b in ((t["k"], c["k"]), (t["v"], c["v"])):
        assert np.array_equal(a.cpu().numpy().view(np.uint16), b.view(np.uint16))
    assert np.array_equal(t["weight"].cpu().numpy(), c["weight"]) and ops.device_status() == 0


def test_decode_evict_append_run(cuda):
    """A bounded cache in use: steps of append, decode (weights accumulate)
    and, whenever the cache is full, eviction back to the budget, over a shared
    prefix; the caches, weights and positions follow the 64-bit restatement's
    selection (made on the device's weights, so that no rounding decides)."""
    import torch
    from leaninfer_b200 import ops
    from oracle import kv
    r = rng(800)
    B, P, ctx, Hkv, G, budget = 3, 150, 24, 2, 4, 16
    c, t, cache = _cache(r, cuda, B, ctx, Hkv, [0] * B, P, stale=3.0)
    t["weight"].zero_()
    kw = dict(head_dim=128, rope_dim=64, layout="half", theta=1e6)
    R = ops.Rope(**kw)
    n = 0
    host = {a: t[a].cpu().numpy() for a in ("k", "v", "weight", "slot_pos")}
    for step in range(45):
        n += 1
        t["lens"].fill_(n)
        pos = np.full(B, P + step, np.int32)
        q, k, v = (T(r.standard_normal((B, h, 128)).astype(np.float32), cuda) for h in (Hkv * G, Hkv, Hkv))
        qr = cache.append(k, v, T(pos, cuda), q=q, rope=R)
        out = cache.decode(qr)
        host["k"][:, n - 1] = t["k"][:, n - 1].cpu().numpy()
        host["v"][:, n - 1] = t["v"][:, n - 1].cpu().numpy()
        host["slot_pos"][:, :, n - 1] = pos[:, None]
        ref, _ = kv.attn(qr.double().cpu().numpy(), host["k"], host["v"], [n] * B, c["kp"], c["vp"])
        assert np.linalg.norm(out.double().cpu().numpy() - ref) <= 1e-5 * np.linalg.norm(ref)
        host["weight"] = t["weight"].cpu().numpy()
        # per kv head the q heads' probabilities on own slots: the weights of a step sum to less than G
        if n == ctx:
            cache.evict(T(pos, cuda), budget, n_sink=2, n_recent=5)
            lens = np.full(B, n)
            kv.evict(host["k"], host["v"], host["weight"], host["slot_pos"], lens, pos, budget, P + 2, 5)
            n = budget
            for a in ("k", "v", "weight", "slot_pos"):
                assert np.array_equal(t[a].cpu().numpy(), host[a]), (step, a)
            assert t["lens"].tolist() == [budget] * B
            kept = host["slot_pos"][:, :, :n]
            assert (kept < P + 2).sum() == B * Hkv * 2 and (kept > pos[0] - 5).sum() == B * Hkv * 5
    assert ops.device_status() == 0


# --------------------------------------------------------------------------
@pytest.mark.parametrize("dt,head_dim,rope_dim,heads,layout", [
    ("f32", 8, 8, 1, "half"), ("f32", 16, 8, 1, "interleaved"), ("bf16", 16, 8, 1, "half"), ("bf16", 2, 2, 2, "half"),
    ("f16", 2, 2, 1, "interleaved"), ("bf16", 32, 0, 1, "half"), ("f16", 8, 4, 3, "interleaved"),
    ("f32", 48, 12, 1, "half")])
def test_rope_of_small_heads_over_many_tokens(cuda, dt, head_dim, rope_dim, heads, layout):
    """One to three small heads a token: blocks take hundreds of tokens, which
    is more tokens than a block has threads."""
    from leaninfer_b200 import ops
    from oracle import kv
    r = rng(900 + head_dim + heads)
    tokens = 260011
    kw = dict(head_dim=head_dim, rope_dim=rope_dim, layout=layout, theta=1e4)
    x = T(r.standard_normal((tokens, heads, head_dim)).astype(np.float32), cuda).to(_torch_dt(dt))
    pos = r.integers(0, 1 << 20, tokens).astype(np.int32)
    x64 = x.double().cpu().numpy()
    R = ops.Rope(**kw)
    _check_rope(ops.rope(R, x, T(pos, cuda)), kv.rope(x64, pos, **kw), x64, 1.0, dt)
    _check_rope(ops.rope(R, x, T(pos, cuda), out=x), kv.rope(x64, pos, **kw), x64, 1.0, dt, "in place")
    assert ops.device_status() == 0


@pytest.mark.parametrize("kw", [dict(q_scale=1e38, scale=1.2e-38, k_scale=0.05),
                                dict(q_scale=1e38, scale=-1.2e-38, k_scale=0.05),
                                dict(q_scale=1e-40, scale=1e37, k_scale=500.0)])
@pytest.mark.parametrize("B,P", [(3, 50), (20, 1700)])
def test_queries_at_the_ends_of_fp32(cuda, B, P, kw):
    """Rows of q whose largest value is beyond 2^127, or below the normal
    floats, with scales that leave ordinary scores (30 at most): the row's
    power of two and its inverse stay exact."""
    class Clipped:                         # fp32's largest is 3.4e38
        def __init__(self):
            self.r = rng(910)

        def __getattr__(self, name):
            return getattr(self.r, name)

        def standard_normal(self, shape):
            return np.clip(self.r.standard_normal(shape), -3.3, 3.3)

    _attn_check(cuda, Clipped(), B, P, 70, [(i * 13) % 71 for i in range(B)], 2, 5, **kw)


def test_evict_workspace_does_not_grow_with_budgets(cuda):
    """One workspace serves every budget: a host that varies it allocates no
    more, and the address that a captured eviction holds stays in use."""
    import gc

    import torch
    r = rng(920)
    c, t, cache = _cache(r, cuda, 2, 600, 2, [600, 600], stale=None)
    pos = T(np.full(2, 599, np.int32), cuda)
    cache.evict(pos, 599)
    gc.collect()                           # what earlier tests left is not freed in between
    before = torch.cuda.memory_allocated()
    for budget in (590, 580, 400, 301, 300, 299, 200, 100, 7, 0):
        cache.evict(pos, budget)
        assert t["lens"].tolist() == [budget] * 2
        assert torch.cuda.memory_allocated() == before


# --------------------------------------------------------------------------
@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("pad", [0, 8, 12, 2, 1])
def test_append_with_every_vector_width(cuda, dt, layout, pad):
    """Prompts of 700 tokens out of projections whose row length allows
    vectors of 8, 4, 2 or 1 values: blocks of several tokens, several rounds,
    and tokens split over the heads."""
    from leaninfer_b200 import ops
    from oracle import kv
    r = rng(930 + pad)
    B, ctx, Hkv, G, each = 3, 710, 3, 4, 700
    c, t, cache = _cache(r, cuda, B, ctx, Hkv, [705, 700, 710], stale=None)
    kw = dict(head_dim=128, rope_dim=64 if layout == "half" else 128, layout=layout, theta=1e6)
    first = np.array([5, 0, 10])
    seq, slot = np.repeat(np.arange(B), each), (first[:, None] + np.arange(each)).reshape(-1)
    n = B * each
    pos = (slot + 1000).astype(np.int32)
    proj = T(r.standard_normal((n, (G + 2) * Hkv * 128 + pad)).astype(np.float32), cuda).to(_torch_dt(dt))
    cut = lambda a, b: proj[:, a * 128:b * 128].view(n, b - a, 128)
    q, k, v = cut(0, G * Hkv), cut(G * Hkv, (G + 1) * Hkv), cut((G + 1) * Hkv, (G + 2) * Hkv)
    got = cache.append(k, v, T(pos, cuda), q=q, rope=ops.Rope(**kw), seq=T(seq.astype(np.int32), cuda),
                       slot=T(slot.astype(np.int32), cuda))
    q64, k64, v64 = (a.double().cpu().numpy() for a in (q, k, v))
    _check_rope(got, kv.rope(q64, pos, **kw), q64, 1.0, dt, "q")
    k_ref = kv.rope(k64, pos, **kw)
    kc, vc = t["k"].cpu().numpy(), t["v"].cpu().numpy()
    tol = 2.0 ** -20 * np.abs(k64).max() + 2.0 ** -25
    assert np.all(np.abs(kc[seq, slot].astype(np.float64) - k_ref) <= tol + 2.0 ** -11 * np.abs(k_ref))
    assert np.all(np.abs(vc[seq, slot].astype(np.float64) - v64) <= 2.0 ** -11 * np.abs(v64) + 2.0 ** -25)
    rest = np.ones((B, ctx), bool)
    rest[seq, slot] = False
    assert np.array_equal(kc[rest], c["k"][rest]) and np.array_equal(vc[rest], c["v"][rest])
    w, sp = t["weight"].cpu().numpy(), t["slot_pos"].cpu().numpy()
    assert np.all(w[seq, :, slot] == 0) and np.all(sp[seq, :, slot] == pos[:, None])
    rest_h = np.broadcast_to(rest[:, None], w.shape)
    assert np.array_equal(w[rest_h], c["weight"][rest_h]) and np.array_equal(sp[rest_h], c["slot_pos"][rest_h])
    assert ops.device_status() == 0


@pytest.mark.parametrize("B,P", [(4500, 13), (4500, 100), (2049, 29)])
def test_many_sequences_over_a_prefix(cuda, B, P):
    """More sequences than the length scan has entries, over a prefix that goes
    with the own tokens (4500 x 13 x 512 bytes are below 30 MB) and over one
    that the tensor-core kernel takes."""
    r = rng(940 + P)
    lens = r.integers(0, 6, B).astype(np.int32)
    lens[100:1300] = 0
    _attn_check(cuda, r, B, P, 5, lens, 1, 2, decay=0.5)


@pytest.mark.parametrize("B,P,ctx,limit", [(8, 131072, 16, 4e-6), (16, 0, 32768, 2.5e-6)])
def test_long_sums_stay_as_exact_as_fp32(cuda, B, P, ctx, limit):
    """Sums over many tokens, normwise against 64 bits. The tensor cores round
    towards zero, half a unit (2^-24 of the sum at most) a product on average;
    what that adds up to is bounded by how long a sum stays with them.
      prefix  64 products (4 tiles of 128 tokens, hi and lo parts, 16 tokens
              each) to a sum, whose partial sums have 2/3 of its size on
              average: 64 * 2^-24 * 2/3 = 2.5e-6. The score's 8 hi products:
              8 * 2^-24 * 1.5 (q's size) = 7e-7. Limit 4e-6; a sum left alone over
              a block's 28 tiles would be off by 1.8e-5.
      own     16 steps to a sum: 16 * 2^-24 * 2/3 = 6.4e-7, scores 7e-7, the
              split of p 2^-23. Limit 2.5e-6; left alone over a warp's 221 steps:
              8.8e-6.
    """
    import torch
    from leaninfer_b200 import ops
    Hkv, G = 8, 4
    g = torch.Generator(device=cuda).manual_seed(950 + B)
    n16 = lambda *s: torch.randn(*s, generator=g, device=cuda, dtype=torch.float16)
    k, v = n16(B, ctx, Hkv, 128), n16(B, ctx, Hkv, 128)
    kp, vp = (n16(P, Hkv, 128), n16(P, Hkv, 128)) if P else (None, None)
    q = 1.5 * torch.randn(B, Hkv * G, 128, generator=g, device=cuda)
    cache = ops.KVCache(k, v, torch.full((B,), ctx, device=cuda, dtype=torch.int32), k_prefix=kp, v_prefix=vp)
    got = cache.decode(q).double()
    ref = torch.empty_like(got)
    for s in range(B):
        for j in range(Hkv):
            kk, vv = ((torch.cat([p[:, j], o[s, :, j]]) if P else o[s, :, j]).double() for p, o in ((kp, k), (vp, v)))
            sc = q[s, j * G:(j + 1) * G].double() @ kk.T * 128 ** -0.5
            ref[s, j * G:(j + 1) * G] = sc.softmax(-1) @ vv
    err = float((got - ref).norm() / ref.norm())
    assert err <= limit, f"{err:.2e}"
    assert ops.device_status() == 0


@pytest.mark.parametrize("P", [100, 3000])
def test_first_calls_inside_a_capture(cuda, P):
    """Append, decode and evict of a cache that has made no call yet, captured
    (the workspaces come from the capture's pool), replayed and then called
    eagerly with other work in between: the bits of eager calls alone."""
    import torch
    from leaninfer_b200 import ops
    r = rng(960)
    B, ctx, Hkv, G, budget = 12, 40, 2, 4, 30
    R = ops.Rope(head_dim=128, rope_dim=64, theta=1e6)
    c, t, _ = _cache(r, cuda, B, ctx, Hkv, [36] * B, P, stale=None)
    q, k, v = (T(r.standard_normal((B, h, 128)).astype(np.float32), cuda) for h in (Hkv * G, Hkv, Hkv))
    pos = T(np.full(B, P + 36, np.int32), cuda)

    def fresh():
        d = {n: x.clone() for n, x in t.items()}
        cache = ops.KVCache(d["k"], d["v"], d["lens"], k_prefix=d["kp"], v_prefix=d["vp"], weight=d["weight"],
                            slot_pos=d["slot_pos"])
        return d, cache, torch.zeros_like(q), torch.zeros_like(q)

    def run(d, cache, qr, out):
        cache.append(k, v, pos, q=q, rope=R, q_out=qr)
        cache.decode(qr, out=out)
        cache.evict(pos, budget, n_sink=2, n_recent=4)

    eager, graphed = fresh(), fresh()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run(*graphed)
    for turn in range(3):
        run(*eager)
        noise = [torch.randn(1 << 20, device=cuda) for _ in range(4)]      # what the allocator hands out now
        if turn == 2:
            run(*graphed)
        else:
            graph.replay()
        del noise
        for name in t:
            assert torch.equal(eager[0][name], graphed[0][name]), (turn, name)
        assert torch.equal(eager[3], graphed[3])
    assert ops.device_status() == 0


def test_repeated_sources(cuda):
    """Sources may repeat: one q for every sequence, one head for every head."""
    import torch
    from leaninfer_b200 import ops
    r = rng(970)
    R = ops.Rope(head_dim=64, rope_dim=32, theta=1e5)
    one = T(r.standard_normal((1, 1, 64)).astype(np.float32), cuda)
    pos = T(np.arange(9, dtype=np.int32), cuda)
    assert torch.equal(ops.rope(R, one.expand(9, 5, 64), pos), ops.rope(R, one.expand(9, 5, 64).contiguous(), pos))
    with pytest.raises(ops.LeanInferError):
        ops.rope(R, torch.zeros(9, 5, 64, device=cuda), pos, out=one.expand(9, 5, 64).clone()[:1].expand(9, 5, 64))
    for B, P in ((4, 20), (20, 2000)):
        c, t, cache = _cache(r, cuda, B, 30, 2, [30] * B, P)
        q = T(r.standard_normal((1, 8, 128)).astype(np.float32), cuda).expand(B, 8, 128)
        assert torch.equal(cache.decode(q, decay=0.0), cache.decode(q.contiguous(), decay=0.0))
    assert ops.device_status() == 0


def test_launches_follow_the_current_stream(cuda):
    """The stream handle that the wrappers pass is the current stream's."""
    import torch
    from leaninfer_b200 import ops
    assert ops._stream() == torch.cuda.current_stream().cuda_stream
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        assert ops._stream() == side.cuda_stream != torch.cuda.default_stream().cuda_stream
    x = torch.zeros(1, device=cuda)
    with torch.cuda.graph(torch.cuda.CUDAGraph()):
        x += 1
        assert ops._stream() == torch.cuda.current_stream().cuda_stream
