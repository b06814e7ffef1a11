"""Argument checks of the KV-cache entries and of their Python wrappers: every
refusal happens on the host before any CUDA call, so these run without a GPU."""
from __future__ import annotations

import ctypes

import pytest

from conftest import ROOT

BAD_ARG, BAD_SHAPE, UNSUPPORTED, WORKSPACE, MISALIGNED = 2001, 2002, 2003, 2004, 2005
P = 4096                                   # an address nothing dereferences


@pytest.fixture(scope="module")
def lib():
    from leaninfer_b200 import _lib, build
    build.build()
    return _lib.load()


def _cache(**kw):
    from leaninfer_b200._lib import KvCache
    d = dict(n_seqs=4, max_ctx=64, n_kv_heads=2, head_dim=128, k=P, v=P, len=P, weight=P, slot_pos=P)
    d.update(kw)
    return KvCache(**d)


def _rope(**kw):
    from leaninfer_b200._lib import RopeParams
    d = dict(layout=1, head_dim=128, rope_dim=64, theta=1e4, freq_scale=1.0, attn_factor=1.0)
    d.update(kw)
    return RopeParams(**d)


def test_struct_layouts_match_c(tmp_path):
    import subprocess
    from leaninfer_b200._lib import KvCache, RopeParams
    src = tmp_path / "t.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "leaninfer-cuda.h"\nint main(void){'
                   'printf("%zu %zu %zu %zu %zu %zu\\n", sizeof(li_rope), offsetof(li_rope, theta),'
                   'offsetof(li_rope, freq_factors), sizeof(li_kv_cache), offsetof(li_kv_cache, n_prefix),'
                   'offsetof(li_kv_cache, slot_pos)); return 0;}\n')
    exe = tmp_path / "t"
    r = subprocess.run(["gcc", "-std=c99", "-Wall", "-Werror", f"-I{ROOT / 'include'}", str(src), "-o", str(exe)],
                       capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    got = [int(v) for v in subprocess.run([str(exe)], capture_output=True, text=True).stdout.split()]
    assert got == [ctypes.sizeof(RopeParams), RopeParams.theta.offset, RopeParams.freq_factors.offset,
                   ctypes.sizeof(KvCache), KvCache.n_prefix.offset, KvCache.slot_pos.offset]


@pytest.mark.parametrize("change,dtype,want", [
    (dict(layout=2), 0, UNSUPPORTED), (dict(head_dim=127), 0, BAD_SHAPE), (dict(head_dim=0), 0, BAD_SHAPE),
    (dict(head_dim=514), 0, BAD_SHAPE), (dict(rope_dim=130), 0, BAD_SHAPE), (dict(rope_dim=33), 0, BAD_SHAPE),
    (dict(rope_dim=-2), 0, BAD_SHAPE), (dict(theta=1.0), 0, BAD_ARG), (dict(theta=float("nan")), 0, BAD_ARG),
    (dict(theta=float("inf")), 0, BAD_ARG), (dict(freq_scale=0.0), 0, BAD_ARG),
    (dict(freq_scale=float("inf")), 0, BAD_ARG), (dict(attn_factor=float("nan")), 0, BAD_ARG),
    (dict(ext_factor=1.0), 0, BAD_ARG), (dict(ext_factor=1.0, n_ctx_orig=4096, beta_fast=0.0), 0, BAD_ARG),
    (dict(ext_factor=1.0, n_ctx_orig=4096, beta_fast=32.0, beta_slow=-1.0), 0, BAD_ARG),
    (dict(freq_factors=P + 2), 0, MISALIGNED), (dict(), 8, UNSUPPORTED), (dict(), 31, UNSUPPORTED)])
def test_rope_parameters(lib, change, dtype, want):
    R = _rope(**change)
    assert lib.li_launch_rope(ctypes.byref(R), dtype, P, P, P, 2, 3, 384, 128, 384, 128, 0, None) == want


def test_rope_pointers(lib):
    R = ctypes.byref(_rope())
    f = lib.li_launch_rope
    st = (384, 128, 384, 128, 0, None)
    assert f(None, 0, P, P, P, 2, 3, *st) == BAD_ARG
    assert f(R, 0, None, P, P, 2, 3, *st) == BAD_ARG
    assert f(R, 0, P, None, P, 2, 3, *st) == BAD_ARG
    assert f(R, 0, P, P, None, 2, 3, *st) == BAD_ARG
    assert f(R, 0, P, P, P, -1, 3, *st) == BAD_ARG
    assert f(R, 0, P + 2, P, P, 2, 3, *st) == MISALIGNED
    assert f(R, 1, P + 1, P, P, 2, 3, *st) == MISALIGNED
    assert f(R, 0, P, P, P + 2, 2, 3, *st) == MISALIGNED
    assert f(R, 0, P, P, P, 0, 3, *st) == 0 and f(R, 0, P, P, P, 2, 0, *st) == 0


CACHE_FAULTS = [
    (dict(k=None), BAD_ARG), (dict(v=None), BAD_ARG), (dict(len=None), BAD_ARG), (dict(n_seqs=-1), BAD_ARG),
    (dict(max_ctx=0), BAD_ARG), (dict(n_kv_heads=0), BAD_ARG), (dict(n_prefix=-1), BAD_ARG),
    (dict(n_prefix=3, k_prefix=P), BAD_ARG), (dict(n_prefix=3, v_prefix=P), BAD_ARG), (dict(head_dim=64), UNSUPPORTED),
    (dict(k=P + 8), MISALIGNED), (dict(v=P + 8), MISALIGNED), (dict(n_prefix=3, k_prefix=P + 8, v_prefix=P), MISALIGNED),
    (dict(n_prefix=3, k_prefix=P, v_prefix=P + 8), MISALIGNED), (dict(len=P + 2), MISALIGNED),
    (dict(weight=P + 2), MISALIGNED), (dict(slot_pos=P + 1), MISALIGNED),
    (dict(n_seqs=1 << 20, n_kv_heads=1 << 11), BAD_SHAPE)]


@pytest.mark.parametrize("change,want", CACHE_FAULTS)
def test_cache_descriptor(lib, change, want):
    C = ctypes.byref(_cache(**change))
    assert lib.li_launch_kv_append(C, None, 0, None, 0, None, 0, 0, P, 256, P, 256, P, None, None, 2, None) == want
    assert lib.li_launch_attn_kv_decode(C, P, 512, 4, 0.1, P, 1.0, P, 1 << 40, None) == want
    assert lib.li_launch_kv_evict(C, P, 8, 0, 0, P, 1 << 40, None) == want
    assert lib.li_attn_kv_workspace_size(C, 4) == 0
    assert lib.li_kv_evict_workspace_size(C, 8) == 0


def test_append_arguments(lib):
    C, R = ctypes.byref(_cache()), ctypes.byref(_rope())
    f = lib.li_launch_kv_append
    ok = dict(C=C, R=R, dtype=0, q=P, qs=512, qo=P, qos=512, hq=4, k=P, ks=256, v=P, vs=256, pos=P, seq=None, slot=None,
              n=2)

    def call(**kw):
        return f(*{**ok, **kw}.values(), None)

    assert call(C=None) == BAD_ARG
    assert call(k=None) == BAD_ARG and call(v=None) == BAD_ARG and call(pos=None) == BAD_ARG
    assert call(n=-1) == BAD_ARG and call(qo=None) == BAD_ARG and call(hq=0) == BAD_ARG
    assert call(dtype=12) == UNSUPPORTED
    assert call(n=5) == BAD_SHAPE                                   # five tokens, four sequences, no seq
    assert call(R=ctypes.byref(_rope(head_dim=64))) == BAD_SHAPE
    assert call(R=ctypes.byref(_rope(layout=7))) == UNSUPPORTED
    assert call(k=P + 2) == MISALIGNED and call(seq=P + 1) == MISALIGNED and call(slot=P + 2) == MISALIGNED
    assert call(n=0) == 0


def test_decode_arguments(lib):
    c = _cache(n_prefix=100, k_prefix=P, v_prefix=P)
    C = ctypes.byref(c)
    need = lib.li_attn_kv_workspace_size(C, 8)
    assert need > 0
    ok = dict(C=C, q=P, qs=1024, hq=8, scale=0.1, out=P, decay=1.0, ws=P, wb=need)

    def call(**kw):
        return lib.li_launch_attn_kv_decode(*{**ok, **kw}.values(), None)

    assert call(q=None) == BAD_ARG and call(out=None) == BAD_ARG and call(hq=0) == BAD_ARG
    assert call(decay=-0.5) == BAD_ARG and call(decay=float("nan")) == BAD_ARG and call(decay=float("inf")) == BAD_ARG
    assert call(scale=float("nan")) == BAD_ARG and call(scale=float("-inf")) == BAD_ARG
    assert call(hq=7) == BAD_SHAPE and call(hq=34) == UNSUPPORTED
    assert call(q=P + 4) == MISALIGNED and call(out=P + 8) == MISALIGNED and call(qs=1023) == MISALIGNED
    assert call(ws=None) == WORKSPACE and call(wb=need - 1) == WORKSPACE and call(ws=P + 8) == MISALIGNED
    c.n_seqs = 0
    assert call() == 0


def test_evict_arguments(lib):
    c = _cache()
    C = ctypes.byref(c)
    need = lib.li_kv_evict_workspace_size(C, 48)
    assert need > 0 and lib.li_kv_evict_workspace_size(C, 65) == 0 and lib.li_kv_evict_workspace_size(C, -1) == 0
    ok = dict(C=C, pos=P, budget=48, sink=4, recent=16, ws=P, wb=need)

    def call(**kw):
        return lib.li_launch_kv_evict(*{**ok, **kw}.values(), None)

    assert call(pos=None) == BAD_ARG and call(budget=-1) == BAD_ARG
    assert call(sink=-1) == BAD_ARG and call(recent=-1) == BAD_ARG
    assert call(budget=65) == BAD_SHAPE and call(sink=40) == BAD_SHAPE and call(sink=2**31 - 1) == BAD_SHAPE
    assert call(ws=None) == WORKSPACE and call(wb=need - 1) == WORKSPACE and call(ws=P + 4) == MISALIGNED
    assert call(pos=P + 2) == MISALIGNED
    for gone in ("weight", "slot_pos"):
        d = _cache(**{gone: None})
        assert call(C=ctypes.byref(d)) == BAD_ARG
    c.n_seqs = 0
    assert call() == 0


def test_wrappers_refuse_cpu_tensors_and_wrong_shapes(lib):
    import torch
    from leaninfer_b200 import ops
    r = ops.Rope(head_dim=128, rope_dim=64)
    x, pos = torch.zeros(2, 3, 128), torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        ops.rope(r, x, pos)
    with pytest.raises(ValueError, match="128"):
        ops.rope(r, torch.zeros(2, 3, 64), pos)
    with pytest.raises(ValueError, match="fp32, fp16"):
        ops.rope(r, x.double(), pos)
    with pytest.raises(ValueError, match="layout"):
        ops.Rope(head_dim=128, layout="quarter")
    k = torch.zeros(2, 8, 2, 128, dtype=torch.float16)
    n = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        ops.KVCache(k, k.clone(), n)
    with pytest.raises(ValueError, match="fp16"):
        ops.KVCache(k.float(), k.float(), n)
    with pytest.raises(ValueError, match="shape"):
        ops.KVCache(k, k[:, :4], n)
    with pytest.raises(ValueError, match="together"):
        ops.KVCache(k, k.clone(), n, k_prefix=k[0])
    with pytest.raises(ValueError, match="weight"):
        ops.KVCache(k, k.clone(), n, weight=torch.zeros(2, 2, 7))


def _layer(**kw):
    from leaninfer_b200._lib import AttnLayer
    d = dict(hidden=1024, n_q_heads=8, n_kv_heads=2, head_dim=128, rope_dim=64, w_in_type=12, w_out_type=12,
             rope_theta=1e6, in_norm_eps=1e-6, qk_norm_eps=1e-6, w_in=P, w_out=P)
    d.update(kw)
    return AttnLayer(**d)


def test_layer_on_a_managed_cache_arguments(lib):
    c = _cache()
    need = lib.li_attn_layer_kv_workspace_size(ctypes.byref(_layer()), ctypes.byref(c))
    assert need > lib.li_attn_kv_workspace_size(ctypes.byref(c), 8) > 0

    def call(L=None, R=None, C=c, x=P, y=P, pos=P, decay=1.0, ws=P, wb=need):
        return lib.li_launch_attn_layer_decode_kv(ctypes.byref(L or _layer()), ctypes.byref(R) if R else None,
                                                  ctypes.byref(C), x, y, pos, decay, ws, wb, None)

    for change, want in ((dict(w_in=None), BAD_ARG), (dict(w_out=None), BAD_ARG), (dict(head_dim=64), UNSUPPORTED),
                         (dict(n_kv_heads=4), BAD_SHAPE), (dict(n_q_heads=7), BAD_SHAPE), (dict(n_q_heads=34), UNSUPPORTED),
                         (dict(w_in_type=2), UNSUPPORTED), (dict(w_out_type=0), UNSUPPORTED), (dict(rope_dim=63), BAD_SHAPE),
                         (dict(rope_theta=0.5), BAD_ARG), (dict(in_norm_w=P + 4), MISALIGNED)):
        assert call(L=_layer(**change)) == want, change
    assert call(x=None) == BAD_ARG and call(y=None) == BAD_ARG and call(pos=None) == BAD_ARG
    assert call(decay=-1.0) == BAD_ARG and call(decay=float("inf")) == BAD_ARG
    assert call(R=_rope(head_dim=64)) == BAD_SHAPE and call(R=_rope(theta=0.0)) == BAD_ARG
    assert call(x=P + 4) == MISALIGNED and call(pos=P + 2) == MISALIGNED and call(ws=P + 8) == MISALIGNED
    assert call(ws=None) == WORKSPACE and call(wb=need - 1) == WORKSPACE
    for change, want in CACHE_FAULTS:
        assert call(C=_cache(**change)) == want, change
    c.n_seqs = 0
    assert call() == 0


def test_rope_node_checks(lib):
    """The ggml ROPE node's checks; a node that passes them reaches the entry's
    own (here: a head_dim beyond its limit)."""
    from leaninfer_b200 import ggml
    from leaninfer_b200._lib import GgmlTensor

    def t(kind, ne, es):
        d = GgmlTensor()
        d.type, d.data = kind, P
        s = es
        for i in range(4):
            d.ne[i] = ne[i] if i < len(ne) else 1
            d.nb[i] = s
            s *= d.ne[i]
        return d

    def run(x=None, pos=None, ff=None, out=None, **kw):
        p = [0, kw.get("dims", 64), kw.get("mode", 2), 0, 4096, 1e4, 1.0, 0.0, 1.0, 32.0, 1.0]
        x = x or t(ggml.F32, [128, 4, 5], 4)
        nd = ggml.node(ggml.OP_ROPE, out or t(x.type, list(x.ne), x.nb[0]), [x, pos or t(ggml.I32, [5], 4), ff], p)
        return lib.li_ggml_compute_forward(ctypes.byref(nd), None, 0, None)

    assert run(mode=1) == UNSUPPORTED and run(mode=8) == UNSUPPORTED
    assert run(x=t(ggml.Q8_0, [128, 4, 5], 34)) == UNSUPPORTED
    assert run(pos=t(ggml.F32, [5], 4)) == UNSUPPORTED
    assert run(out=t(ggml.F16, [128, 4, 5], 2)) == UNSUPPORTED
    assert run(pos=t(ggml.I32, [4], 4)) == BAD_SHAPE
    assert run(x=t(ggml.F32, [128, 4, 5, 2], 4)) == BAD_SHAPE
    assert run(out=t(ggml.F32, [128, 4, 6], 4)) == BAD_SHAPE
    assert run(ff=t(ggml.F32, [64], 4)) == BAD_SHAPE
    odd = t(ggml.F32, [128, 4, 5], 4)
    odd.nb[1] += 2
    assert run(x=odd) == BAD_SHAPE
    assert run(dims=130) == BAD_SHAPE and run(x=t(ggml.F32, [514, 4, 5], 4)) == BAD_SHAPE
    gone = t(ggml.I32, [5], 4)
    gone.data = None
    assert run(pos=gone) == BAD_ARG


class _On:
    """Stands for a CUDA tensor of a device; nothing reads it."""

    def __init__(self, index, shape=(), dtype=None):
        self.index, self.shape, self.dtype = index, shape, dtype

    def get_device(self):
        return self.index


def test_layer_step_refuses_tensors_of_another_device(monkeypatch):
    """Every tensor that a layer step on a managed cache reads: the step's own,
    the frequency divisors and the layer's weights."""
    import types

    import torch
    from leaninfer_b200 import ops
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    monkeypatch.setattr(ops._lib, "load", lambda: pytest.fail("the call went past the device check"))
    cache = types.SimpleNamespace(index=0, n_seqs=2)

    def step(where):
        at = lambda name: 1 if name == where else 0
        layer = object.__new__(ops.AttnLayerDecode)
        layer.L = types.SimpleNamespace(hidden=64)
        layer.keep = [_On(at(n)) if n else None for n in ("w_in", "w_out", "", "q_norm_w", "")]
        rope = types.SimpleNamespace(keep=_On(at("freq_factors")))
        x, y = (_On(at(n), (2, 64), torch.float32) for n in ("x", "y"))
        layer.step_kv(x, y, cache, _On(at("pos")), rope=rope, workspace=_On(at("workspace")))

    for where in ("x", "y", "pos", "workspace", "freq_factors", "w_in", "w_out", "q_norm_w"):
        with pytest.raises(ValueError, match="one device"):
            step(where)


@pytest.mark.parametrize("n_seqs,heads,ctx", [(1 << 15, 1 << 10, 1 << 15), (1 << 20, 1, 1 << 20),
                                              ((1 << 31) - 1, 1, (1 << 31) - 1), (1, (1 << 31) - 1, (1 << 31) - 1)])
def test_cache_counts_beyond_the_size_arithmetic(lib, n_seqs, heads, ctx):
    """2^40 and more (sequence, kv head, slot) triples are refused, before any
    product of them is a size: at the last two, a workspace of 2^64 bytes."""
    C = ctypes.byref(_cache(n_seqs=n_seqs, n_kv_heads=heads, max_ctx=ctx))
    assert lib.li_kv_evict_workspace_size(C, (ctx + 1) // 2) == 0 == lib.li_attn_kv_workspace_size(C, heads)
    assert lib.li_launch_kv_evict(C, P, (ctx + 1) // 2, 0, 0, P, 1 << 62, None) == BAD_SHAPE
    assert lib.li_launch_attn_kv_decode(C, P, 128, heads, 0.1, P, 1.0, P, 1 << 62, None) == BAD_SHAPE
    assert lib.li_launch_kv_append(C, None, 0, None, 0, None, 0, 0, P, 128, P, 128, P, None, None, 0, None) == BAD_SHAPE


def test_outputs_whose_rows_overlap(lib):
    """A destination whose rows lie on one another (an expanded tensor, say)
    would be written by several threads at once; sources may repeat."""
    R, C = ctypes.byref(_rope()), ctypes.byref(_cache())

    def rope(n, heads, ts, hs):
        return lib.li_launch_rope(R, 0, P, P, P, n, heads, 0, 0, ts, hs, 0, None)

    assert rope(2, 3, 0, 128) == BAD_SHAPE and rope(2, 3, 384, 0) == BAD_SHAPE
    assert rope(2, 3, 127, 256) == BAD_SHAPE and rope(2, 3, 384, -64) == BAD_SHAPE
    assert rope(1, 3, 0, 100) == BAD_SHAPE and rope(9, 1, -100, 0) == BAD_SHAPE

    def append(n, stride):
        return lib.li_launch_kv_append(C, R, 0, P, 512, P, stride, 4, P, 256, P, 256, P, None, None, n, None)

    assert append(2, 0) == BAD_SHAPE and append(3, 511) == BAD_SHAPE and append(2, -384) == BAD_SHAPE
