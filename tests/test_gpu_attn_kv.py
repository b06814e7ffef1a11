"""The attention layer on a managed cache (li_launch_attn_layer_decode_kv) and
the ggml ROPE node, on the GPU.

The layer is held to the framework's oracle of the attention layer, given the
shared prefix as the first tokens of every sequence's cache: the same function
of the same tokens. Tolerances are those of that layer's own parity tests
(test_gpu_attn.py), since the projections' roundings are the same and the
attention adds less: 1e-3 normwise for y with the SIMT projections (up to 2
sequences here), 3e-3 with the tensor-core ones, cache rows 1e-3 and 2e-3.
"""
from __future__ import annotations

import numpy as np
import pytest

from conftest import assert_close, rng

pytestmark = pytest.mark.gpu
BAD_ARG = 2001


def T(a, dev):
    import torch
    return torch.from_numpy(np.ascontiguousarray(a)).to(dev)


def _layer(cuda, w, **kw):
    from leaninfer_b200 import ops
    return ops.AttnLayerDecode(
        hidden=w["hidden"], n_q_heads=w["n_q_heads"], n_kv_heads=w["n_kv_heads"], head_dim=w["head_dim"],
        rope_dim=w["rope_dim"], rope_theta=w["rope_theta"], w_in=T(w["w_in"], cuda), w_out=T(w["w_out"], cuda),
        in_norm_w=T(w["in_norm_w"], cuda), w_in_type=w["wtype"], w_out_type=w["wtype"],
        **({"q_norm_w": T(w["q_norm_w"], cuda), "k_norm_w": T(w["k_norm_w"], cuda)} | kw))


def _f16(u16):
    return np.asarray(u16).view(np.float16).astype(np.float32)


@pytest.mark.parametrize("B,P,ctx,G,wtype", [(1, 0, 40, 5, 12), (2, 130, 60, 4, 8), (9, 300, 50, 5, 12),
                                             (40, 77, 33, 1, 12), (33, 0, 300, 8, 12)])
def test_layer_matches_the_oracle_over_prefix_and_own_tokens(cuda, oracle_mod, B, P, ctx, G, wtype):
    import torch
    from leaninfer_b200 import ops, synth
    r = rng(7000 + B)
    Hkv = 2
    w = synth.attn_layer(r, hidden=1024, n_q_heads=Hkv * G, n_kv_heads=Hkv, rope_dim=32, wtype=wtype)
    layer = _layer(cuda, w)
    L, keep = oracle_mod.make_attn_layer(w)
    lens = np.concatenate([[1], r.integers(1, ctx - 2, B - 1)]).astype(np.int32)
    # the oracle's caches: the prefix in front of every sequence's own slots
    f16 = lambda *s: r.standard_normal(s).astype(np.float16)
    kp, vp = f16(P, Hkv, 128), f16(P, Hkv, 128)
    own_k, own_v = f16(B, ctx, Hkv, 128), f16(B, ctx, Hkv, 128)
    both = lambda p, o: np.ascontiguousarray(np.concatenate([np.broadcast_to(p, (B, *p.shape)), o], 1)).view(np.uint16)
    kc, vc = both(kp, own_k), both(vp, own_v)
    k_d, v_d, len_d = T(own_k, cuda), T(own_v, cuda), T(lens, cuda)
    weight = torch.full((B, Hkv, ctx), 0.5, device=cuda)
    slot_pos = torch.full((B, Hkv, ctx), -1, dtype=torch.int32, device=cuda)
    cache = ops.KVCache(k_d, v_d, len_d, k_prefix=T(kp, cuda) if P else None, v_prefix=T(vp, cuda) if P else None,
                        weight=weight, slot_pos=slot_pos)
    tol_y, tol_row = (1e-3, 1e-3) if B <= 2 else (3e-3, 2e-3)
    for step in range(2):
        x = r.standard_normal((B, 1024)).astype(np.float32)
        pos = (P + lens + step - 1).astype(np.int32)
        len_d.copy_(T(lens + step, cuda))
        y = torch.empty(B, 1024, device=cuda)
        layer.step_kv(T(x, cuda), y, cache, T(pos, cuda), decay=0.0)
        torch.cuda.synchronize()
        y_ref = oracle_mod.attn_layer_decode(L, keep, x, kc, vc, pos)
        assert_close(y.cpu().numpy(), y_ref, tol_y, f"y step {step}")
        at = lens + step - 1
        kg, vg = k_d.cpu().numpy(), v_d.cpu().numpy()
        for s in range(B):
            assert_close(kg[s, at[s]].astype(np.float32), _f16(kc[s, pos[s]]), tol_row, "k row")
            assert_close(vg[s, at[s]].astype(np.float32), _f16(vc[s, pos[s]]), tol_row, "v row")
        wt, sp = weight.cpu().numpy(), slot_pos.cpu().numpy()
        for s in range(B):
            n = lens[s] + step
            # the q heads' probabilities over the own slots: at most G in sum, all of it without a prefix
            assert np.all(wt[s, :, :n] >= 0) and np.all(wt[s, :, n:] == 0.5)
            total = wt[s, :, :n].sum(-1)
            assert np.all(total <= G * 1.00001) and (P > 0 or np.allclose(total, G, rtol=1e-5))
            assert np.all(sp[s, :, n - 1] == pos[s])
    assert ops.device_status() == 0


@pytest.mark.parametrize("layout", ["interleaved", "half"])
def test_layer_equals_its_parts(cuda, layout):
    """With scaled rotary positions: the layer against the projection, append,
    decode, gate and projection called one by one (3 sequences; both sides run
    the same projection kernels, so 1e-5 normwise: the gate's sigmoid and the
    sums' order)."""
    import torch
    from leaninfer_b200 import ops, synth
    r = rng(7100)
    B, P, ctx, Hkv, G = 2, 200, 64, 2, 4
    w = synth.attn_layer(r, hidden=1024, n_q_heads=Hkv * G, n_kv_heads=Hkv, wtype=12)
    layer = _layer(cuda, w, q_norm_w=None, k_norm_w=None)
    R = ops.Rope(head_dim=128, rope_dim=96, layout=layout, theta=1e6, freq_scale=0.25, ext_factor=1.0, n_ctx_orig=4096)
    lens = T(np.array([17, 64], np.int32), cuda)
    make = lambda: [T(r.standard_normal((B, ctx, Hkv, 128)).astype(np.float16), cuda) for _ in range(2)]
    k, v = make()
    kp, vp = (T(r.standard_normal((P, Hkv, 128)).astype(np.float16), cuda) for _ in range(2))
    caches = [ops.KVCache(k.clone(), v.clone(), lens, k_prefix=kp, v_prefix=vp) for _ in range(2)]
    x, pos = T(r.standard_normal((B, 1024)).astype(np.float32), cuda), T(np.array([216, 70000], np.int32), cuda)
    y = layer.step_kv(x, torch.empty(B, 1024, device=cuda), caches[0], pos, rope=R)
    Hq, D = Hkv * G, 128
    proj = ops.rms_norm_matmul_q(12, x, T(w["in_norm_w"], cuda), T(w["w_in"], cuda), 2 * (Hq + Hkv) * D, eps=1e-6)
    cut = lambda a, b: proj[:, a * D:b * D].view(B, b - a, D)
    q = caches[1].append(cut(2 * Hq, 2 * Hq + Hkv), cut(2 * Hq + Hkv, 2 * Hq + 2 * Hkv), pos, q=cut(0, Hq), rope=R)
    o = caches[1].decode(q) * torch.sigmoid(cut(Hq, 2 * Hq))
    ref = ops.rms_norm_matmul_q(12, o.reshape(B, Hq * D), None, T(w["w_out"], cuda), 1024)
    assert_close(y.cpu().numpy(), ref.cpu().numpy(), 1e-5, "y")
    for a, b in zip(caches[0].keep[:2], caches[1].keep[:2]):
        d = (a.float() - b.float()).abs()
        assert float((d > 2.0 ** -10 * b.float().abs() + 1e-6).sum()) == 0            # at most a step of f16
    assert ops.device_status() == 0


def test_bounded_generation_in_a_graph(cuda):
    """Layer steps on a cache that eviction keeps within its budget, the step
    captured once and replayed with lengths and positions advanced on the
    device, the eviction captured too: the same bits as the calls made
    eagerly, and the positions kept are the sinks, the newest and others."""
    import torch
    from leaninfer_b200 import ops, synth
    r = rng(7200)
    B, P, ctx, budget, Hkv, G = 3, 100, 40, 32, 2, 4
    w = synth.attn_layer(r, hidden=1024, n_q_heads=Hkv * G, n_kv_heads=Hkv, wtype=12)
    layer = _layer(cuda, w)
    kp, vp = (T(r.standard_normal((P, Hkv, 128)).astype(np.float16), cuda) for _ in range(2))
    xs = [T(r.standard_normal((B, 1024)).astype(np.float32), cuda) for _ in range(60)]

    def state():
        z = lambda *s, dt=torch.float16: torch.zeros(*s, device=cuda, dtype=dt)
        s = dict(len=z(B, dt=torch.int32), pos=torch.full((B,), P - 1, device=cuda, dtype=torch.int32),
                 x=z(B, 1024, dt=torch.float32), y=z(B, 1024, dt=torch.float32), weight=z(B, Hkv, ctx, dt=torch.float32),
                 slot_pos=z(B, Hkv, ctx, dt=torch.int32), k=z(B, ctx, Hkv, 128), v=z(B, ctx, Hkv, 128))
        s["cache"] = ops.KVCache(s["k"], s["v"], s["len"], k_prefix=kp, v_prefix=vp, weight=s["weight"],
                                 slot_pos=s["slot_pos"])
        return s

    def step(s):
        s["len"].add_(1)
        s["pos"].add_(1)
        layer.step_kv(s["x"], s["y"], s["cache"], s["pos"])

    def shrink(s):
        s["cache"].evict(s["pos"], budget, n_sink=3, n_recent=8)

    eager, graphed = state(), state()
    st = torch.cuda.Stream()
    with torch.cuda.stream(st):
        step(graphed)                       # the workspaces, before the capture
        shrink(graphed)
        for name, t in state().items():
            if name != "cache":
                graphed[name].copy_(t)
        graphs = []
        for f in (step, shrink):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=st):
                f(graphed)
            graphs.append(g)
        n = 0
        for x in xs:
            for s in (eager, graphed):
                s["x"].copy_(x)
            step(eager)
            graphs[0].replay()
            n += 1
            if n == ctx:
                shrink(eager)
                graphs[1].replay()
                n = budget
    st.synchronize()
    for name in ("y", "len", "pos", "weight", "slot_pos", "k", "v"):
        assert torch.equal(eager[name], graphed[name]), name
    assert torch.isfinite(eager["y"]).all() and eager["len"].tolist() == [n] * B
    sp, newest = eager["slot_pos"][:, :, :n].cpu().numpy(), P - 1 + len(xs)
    for s in range(B):
        for j in range(Hkv):
            kept = sorted(sp[s, j])
            assert len(set(kept)) == n and kept[:3] == [P, P + 1, P + 2]
            assert kept[-8:] == list(range(newest - 7, newest + 1))
    assert ops.device_status() == 0


def test_layer_bad_lengths(cuda):
    """Lengths 0 and ctx + 1 append nothing, raise the flag and attend over the
    prefix alone; the other sequence is served."""
    import torch
    from leaninfer_b200 import ops, synth
    r = rng(7300)
    w = synth.attn_layer(r, hidden=1024, n_q_heads=8, n_kv_heads=2, wtype=12)
    layer = _layer(cuda, w)
    k, v = (T(r.standard_normal((3, 16, 2, 128)).astype(np.float16), cuda) for _ in range(2))
    kp, vp = (T(r.standard_normal((40, 2, 128)).astype(np.float16), cuda) for _ in range(2))
    x, pos = T(r.standard_normal((3, 1024)).astype(np.float32), cuda), T(np.array([40, 41, 42], np.int32), cuda)
    outs = []
    for lens in ([0, 5, 17], [0, 5, 0]):
        cache = ops.KVCache(k.clone(), v.clone(), T(np.array(lens, np.int32), cuda), k_prefix=kp, v_prefix=vp)
        outs.append(layer.step_kv(x, torch.empty(3, 1024, device=cuda), cache, pos))
        assert ops.device_status() == BAD_ARG
        assert torch.equal(cache.keep[0][0], k[0]) and torch.equal(cache.keep[0][2], k[2])
        assert not torch.equal(cache.keep[0][1], k[1])
    assert torch.equal(outs[0], outs[1]) and torch.isfinite(outs[0]).all()


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("mode", [0, 2])
def test_rope_node(cuda, dt, mode):
    """The node gives exactly what the entry gives, strided sources included."""
    import torch
    from leaninfer_b200 import ggml, ops
    r = rng(7400)
    dtype = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[dt]
    wide = T(r.standard_normal((9, 6 * 128 + 64)).astype(np.float32), cuda).to(dtype)
    x, pos = wide[:, :768].view(9, 6, 128), T(r.integers(0, 90000, 9).astype(np.int32), cuda)
    ff = T(r.uniform(1, 4, 32).astype(np.float32), cuda)
    out = torch.empty(9, 6, 128, device=cuda, dtype=dtype)
    nd = ggml.node(ggml.OP_ROPE, ggml.desc(out), [ggml.desc(x), ggml.desc(pos), ggml.desc(ff)],
                   [0, 64, mode, 0, 4096, 1e6, 0.25, 1.0, 1.0, 32.0, 1.0])
    assert ggml.compute_forward(nd) == 0
    R = ops.Rope(head_dim=128, rope_dim=64, layout="half" if mode == 2 else "interleaved", theta=1e6, freq_scale=0.25,
                 ext_factor=1.0, n_ctx_orig=4096, freq_factors=ff)
    ref = ops.rope(R, x, pos)
    torch.cuda.synchronize()
    assert torch.equal(out, ref)


def test_layer_step_of_an_empty_batch(cuda):
    """No sequences: nothing happens, as in append, decode and evict."""
    import torch
    from leaninfer_b200 import ops, synth
    w = synth.attn_layer(rng(7500), hidden=1024, n_q_heads=8, n_kv_heads=2, wtype=12)
    layer = _layer(cuda, w)
    z = lambda *s, dt=torch.float32: torch.empty(*s, device=cuda, dtype=dt)
    none = z(0, dt=torch.int32)
    cache = ops.KVCache(z(0, 16, 2, 128, dt=torch.float16), z(0, 16, 2, 128, dt=torch.float16), none)
    y = z(0, 1024)
    assert layer.step_kv(z(0, 1024), y, cache, none) is y
    assert ops.device_status() == 0
