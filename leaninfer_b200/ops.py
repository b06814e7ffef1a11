"""Host-side mirror of the LeanInfer fused-kernel interface on torch tensors.

Each function takes CUDA tensors, calls the matching C-ABI entry of
``libleaninfer_cuda.so`` on torch's current stream and returns the outputs.
Argument meaning follows the reference launchers (cuda/leaninfer-cuda.h,
cuda/leaninfer-fused-ffn.cu, cuda/leaninfer-fused-gate.cu,
cuda/leaninfer-fused-deltanet.cu). PyTorch supplies device memory and
streams only; all arithmetic runs in the library's kernels.
"""
from __future__ import annotations

import ctypes

import numpy as np
import torch

from . import _lib
from ._lib import (LI_DTYPE_BF16, LI_DTYPE_F16, LI_DTYPE_F32, LI_ROPE_HALF, LI_ROPE_INTERLEAVED, LI_WTYPE_Q4_K,
                   LI_WTYPE_Q8_0, AttnLayer, DeltaNetLayer, KvCache, LeanInferError, RopeParams, check)

__all__ = [
    "rms_norm_matmul_f32", "rms_norm_swiglu_f32", "rms_norm_swiglu_f16", "rms_norm_qkv_f32",
    "rms_norm_silu_gate_f32", "deltanet_recurrent_out_f32", "deltanet_recurrent_f32",
    "dequantize", "rms_norm_matmul_q", "rms_norm_qkv_q", "rms_norm_swiglu_q", "ffn_q",
    "DeltaNetLayerDecode", "AttnLayerDecode", "Rope", "rope", "KVCache", "device_status", "row_bytes",
    "LI_WTYPE_Q8_0", "LI_WTYPE_Q4_K",
]


def _stream() -> int:
    # the raw handle of torch.cuda.current_stream(), without building the Stream object around it
    return torch._C._cuda_getCurrentRawStream(torch.cuda.current_device())


def _p(t: torch.Tensor | None) -> int | None:
    if t is None:
        return None
    if not t.is_cuda:
        raise ValueError("LeanInfer kernels take CUDA tensors")
    if not t.is_contiguous():
        raise ValueError("LeanInfer kernels take contiguous tensors")
    return t.data_ptr()


def _legacy_check(what: str) -> None:
    rc = _lib.load().li_get_last_error()
    if rc:
        raise LeanInferError(rc, what)


def row_bytes(wtype: int, k: int) -> int:
    return int(_lib.load().li_row_bytes(wtype, k))


def device_status() -> int:
    """Synchronise and return the device-side status flag (0 = ok)."""
    return int(_lib.load().li_device_status())


# --------------------------------------------------------------------------
# Reference entries
# --------------------------------------------------------------------------
def rms_norm_matmul_f32(x, gamma, W, eps: float = 1e-6):
    N, K = W.shape
    dst = torch.empty(N, device=x.device, dtype=torch.float32)
    _lib.load().li_launch_fused_rms_norm_matmul_f32(_p(x), _p(gamma), _p(W), _p(dst), K, N, eps, _stream())
    _legacy_check("li_launch_fused_rms_norm_matmul_f32")
    return dst


def rms_norm_swiglu_f32(x, gamma, W_gate, W_up, eps: float = 1e-6):
    N, K = W_gate.shape
    h = torch.empty(N, device=x.device, dtype=torch.float32)
    _lib.load().li_launch_fused_rms_norm_swiglu_f32(_p(x), _p(gamma), _p(W_gate), _p(W_up), _p(h),
                                                    K, N, eps, _stream())
    _legacy_check("li_launch_fused_rms_norm_swiglu_f32")
    return h


def rms_norm_swiglu_f16(x, gamma, W_gate, W_up, eps: float = 1e-6):
    N, K = W_gate.shape
    h = torch.empty(N, device=x.device, dtype=torch.float32)
    _lib.load().li_launch_fused_rms_norm_swiglu_f16(_p(x), _p(gamma), _p(W_gate), _p(W_up), _p(h),
                                                    K, N, eps, _stream())
    _legacy_check("li_launch_fused_rms_norm_swiglu_f16")
    return h


def rms_norm_qkv_f32(x, gamma, Ws, eps: float = 1e-6, device_arrays: bool = False):
    """device_arrays: pass W_ptrs / dst_ptrs as arrays in device memory (the
    form the reference's comment prescribes) instead of host arrays."""
    N, K = Ws[0].shape
    outs = [torch.empty(N, device=x.device, dtype=torch.float32) for _ in range(3)]
    if device_arrays:
        wt = torch.tensor([_p(w) for w in Ws], dtype=torch.int64, device=x.device)
        dt = torch.tensor([_p(o) for o in outs], dtype=torch.int64, device=x.device)
        wp = ctypes.cast(ctypes.c_void_p(wt.data_ptr()), ctypes.POINTER(ctypes.c_void_p))
        dp = ctypes.cast(ctypes.c_void_p(dt.data_ptr()), ctypes.POINTER(ctypes.c_void_p))
    else:
        wp = (ctypes.c_void_p * 3)(*[_p(w) for w in Ws])
        dp = (ctypes.c_void_p * 3)(*[_p(o) for o in outs])
    _lib.load().li_launch_fused_rms_norm_qkv_f32(_p(x), _p(gamma), wp, dp, K, N, eps, _stream())
    _legacy_check("li_launch_fused_rms_norm_qkv_f32")
    if device_arrays:
        torch.cuda.current_stream().synchronize()   # the pointer arrays must outlive the launch
    return tuple(outs)


def rms_norm_silu_gate_f32(output, z, gamma, eps: float = 1e-6):
    K = output.shape[-1]
    n_rows = output.numel() // K
    dst = torch.empty_like(output)
    _lib.load().li_launch_fused_rms_norm_silu_gate_f32(_p(output), _p(z), _p(gamma), _p(dst), K, n_rows,
                                                       eps, _stream())
    _legacy_check("li_launch_fused_rms_norm_silu_gate_f32")
    return dst


def deltanet_recurrent_out_f32(q, k, v, g, beta, state_in, W_out, *, head_dim, n_tokens, n_heads,
                               gqa_ratio, repeat_type, n_seqs, hidden_dim, vnb1, vnb2, vnb3):
    """Reference-layout recurrence + projection. Returns (dst, proj_out):
    dst holds per-head outputs then the final state, as in the reference."""
    out_elems = head_dim * n_tokens * n_heads * n_seqs
    dst = torch.empty(out_elems + state_in.numel(), device=q.device, dtype=torch.float32)
    proj = torch.empty(hidden_dim * n_tokens, device=q.device, dtype=torch.float32)
    _lib.load().li_launch_fused_deltanet_recurrent_out_f32(
        _p(q), _p(k), _p(v), _p(g), _p(beta), _p(state_in), _p(W_out), _p(dst), _p(proj),
        head_dim, n_tokens, n_heads, gqa_ratio, repeat_type, n_seqs, hidden_dim, vnb1, vnb2, vnb3,
        _stream())
    _legacy_check("li_launch_fused_deltanet_recurrent_out_f32")
    return dst, proj


# --------------------------------------------------------------------------
# Additive entries
# --------------------------------------------------------------------------
def dequantize(wtype: int, blocks: torch.Tensor, n: int) -> torch.Tensor:
    out = torch.empty(n, device=blocks.device, dtype=torch.float32)
    check(_lib.load().li_launch_dequantize(wtype, _p(blocks), _p(out), n, _stream()), "li_launch_dequantize")
    return out


def rms_norm_matmul_q(wtype, x, gamma, W, N: int, eps: float = 1e-6, out=None):
    n_rows, K = x.shape
    dst = out if out is not None else torch.empty(n_rows, N, device=x.device, dtype=torch.float32)
    check(_lib.load().li_launch_rms_norm_matmul_q(wtype, _p(x), _p(gamma), _p(W), _p(dst), K, N, n_rows,
                                                  eps, _stream()), "li_launch_rms_norm_matmul_q")
    return dst


def rms_norm_qkv_q(wtype, x, gamma, Wq, Wk, Wv, Nq: int, Nk: int, Nv: int, eps: float = 1e-6):
    n_rows, K = x.shape
    q = torch.empty(n_rows, Nq, device=x.device, dtype=torch.float32)
    k = torch.empty(n_rows, Nk, device=x.device, dtype=torch.float32)
    v = torch.empty(n_rows, Nv, device=x.device, dtype=torch.float32)
    check(_lib.load().li_launch_fused_rms_norm_qkv_q(wtype, _p(x), _p(gamma), _p(Wq), _p(Wk), _p(Wv),
                                                     _p(q), _p(k), _p(v), K, Nq, Nk, Nv, n_rows, eps,
                                                     _stream()), "li_launch_fused_rms_norm_qkv_q")
    return q, k, v


def rms_norm_swiglu_q(wtype, x, gamma, Wg, Wu, N: int, eps: float = 1e-6):
    n_rows, K = x.shape
    h = torch.empty(n_rows, N, device=x.device, dtype=torch.float32)
    check(_lib.load().li_launch_fused_rms_norm_swiglu_q(wtype, _p(x), _p(gamma), _p(Wg), _p(Wu), _p(h),
                                                        K, N, n_rows, eps, _stream()),
          "li_launch_fused_rms_norm_swiglu_q")
    return h


def ffn_q(wtype, x, gamma, Wg, Wu, Wd, N: int, eps: float = 1e-6, workspace=None, out=None):
    n_rows, K = x.shape
    lib = _lib.load()
    ws_bytes = int(lib.li_fused_ffn_workspace_size(K, N, n_rows))
    if workspace is None:
        workspace = torch.empty(ws_bytes, device=x.device, dtype=torch.uint8)
    y = out if out is not None else torch.empty(n_rows, K, device=x.device, dtype=torch.float32)
    check(lib.li_launch_fused_ffn_q(wtype, _p(x), _p(gamma), _p(Wg), _p(Wu), _p(Wd), _p(y), K, N, n_rows,
                                    eps, _p(workspace), workspace.numel(), _stream()),
          "li_launch_fused_ffn_q")
    return y


def deltanet_recurrent_f32(q, k, v, g, beta, state_in, *, head_dim, n_tokens, n_heads, gqa_ratio,
                           repeat_type, n_seqs, vnb1, vnb2, vnb3, state_out=None):
    out = torch.empty(n_seqs * n_tokens * n_heads * head_dim, device=q.device, dtype=torch.float32)
    so = state_out if state_out is not None else torch.empty_like(state_in)
    check(_lib.load().li_launch_deltanet_recurrent_f32(
        _p(q), _p(k), _p(v), _p(g), _p(beta), _p(state_in), _p(out), _p(so), head_dim, n_tokens,
        n_heads, gqa_ratio, repeat_type, n_seqs, vnb1, vnb2, vnb3, _stream()),
        "li_launch_deltanet_recurrent_f32")
    return out, so


def deltanet_chunk_prefill_bf16(q, k, v, g, beta, state, scale: float, workspace=None, out=None):
    """Chunked (WY, chunk 64) gated delta rule prefill of one sequence on the
    tensor cores. q, k bf16 [T, Hk, D]; v bf16 [T, Hv, D]; g (log decay), beta
    fp32 [T, Hv]; state fp32 [Hv, D, D] updated in place. Returns o fp32
    [T, Hv, D]."""
    T, Hk, D = q.shape
    Hv = v.shape[1]
    lib = _lib.load()
    ws_bytes = int(lib.li_deltanet_chunk_prefill_workspace_size(T, Hv, D))
    if workspace is None:
        workspace = torch.empty(max(ws_bytes, 16), device=q.device, dtype=torch.uint8)
    o = out if out is not None else torch.empty(T, Hv, D, device=q.device, dtype=torch.float32)
    check(lib.li_launch_deltanet_chunk_prefill_bf16(_p(q), _p(k), _p(v), _p(g), _p(beta), _p(state), _p(o), T, Hk,
                                                    Hv, D, scale, _p(workspace), workspace.numel(), _stream()),
          "li_launch_deltanet_chunk_prefill_bf16")
    return o


def gated_rmsnorm_bf16(o, z, gamma, eps: float = 1e-6):
    """bf16(silu(z) * rmsnorm(o) * gamma) over the last dimension."""
    K = o.shape[-1]
    n = o.numel() // K
    dst = torch.empty(o.shape, device=o.device, dtype=torch.bfloat16)
    check(_lib.load().li_launch_gated_rmsnorm_bf16(_p(o), _p(z), _p(gamma), _p(dst), K, n, eps, _stream()),
          "li_launch_gated_rmsnorm_bf16")
    return dst


def gemm_bf16(A, W, out=None):
    """C (fp32) = A . W^T with A [M, K], W [N, K] bf16, on the tensor cores."""
    M, K = A.shape
    N = W.shape[0]
    C = out if out is not None else torch.empty(M, N, device=A.device, dtype=torch.float32)
    check(_lib.load().li_launch_gemm_bf16_f32(_p(A), _p(W), _p(C), M, N, K, _stream()), "li_launch_gemm_bf16_f32")
    return C


class DeltaNetLayerDecode:
    """One DeltaNet layer's device weights plus a workspace, stepping B
    sequences one token at a time through li_launch_deltanet_layer_decode."""

    def __init__(self, *, hidden, n_k_heads, n_v_heads, head_dim, w_in, conv_w, a_log, dt_bias,
                 norm_w, w_out, w_in_type=LI_WTYPE_Q4_K, w_out_type=LI_WTYPE_Q4_K, in_norm_w=None,
                 in_norm_eps=1e-6, norm_eps=1e-6, l2_eps=1e-6, repeat_type=0, conv_kernel=4):
        self.keep = [w_in, conv_w, a_log, dt_bias, norm_w, w_out, in_norm_w]
        self.L = DeltaNetLayer(
            hidden=hidden, n_k_heads=n_k_heads, n_v_heads=n_v_heads, head_dim=head_dim,
            conv_kernel=conv_kernel, repeat_type=repeat_type, w_in_type=w_in_type,
            w_out_type=w_out_type, in_norm_eps=in_norm_eps, norm_eps=norm_eps, l2_eps=l2_eps,
            in_norm_w=_p(in_norm_w), w_in=_p(w_in), conv_w=_p(conv_w), a_log=_p(a_log),
            dt_bias=_p(dt_bias), norm_w=_p(norm_w), w_out=_p(w_out))
        self.device = w_in.device
        self._ws = None

    @classmethod
    def from_gguf(cls, path, il: int, *, n_k_heads: int, n_v_heads: int, head_dim: int = 128, names=None,
                  device="cuda", **kw) -> "DeltaNetLayerDecode":
        """Layer `il` of a GGUF checkpoint (leaninfer_b200.gguf_file: the
        quantized rows are copied to the device as they are in the file)."""
        from .gguf_file import GGUFFile, deltanet_layer
        with GGUFFile(path) as g:
            w = deltanet_layer(g, il, n_k_heads=n_k_heads, n_v_heads=n_v_heads, head_dim=head_dim, names=names)
        t = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(device)
        return cls(hidden=w["hidden"], n_k_heads=n_k_heads, n_v_heads=n_v_heads, head_dim=head_dim,
                   w_in=t(w["w_in"]), conv_w=t(w["conv_w"]), a_log=t(w["a_log"]), dt_bias=t(w["dt_bias"]),
                   norm_w=t(w["norm_w"]), w_out=t(w["w_out"]), w_in_type=w["wtype"], w_out_type=w["wtype"], **kw)

    @property
    def conv_channels(self) -> int:
        L = self.L
        return 2 * L.n_k_heads * L.head_dim + L.n_v_heads * L.head_dim

    def workspace_bytes(self, n_seqs: int) -> int:
        return int(_lib.load().li_deltanet_layer_workspace_size(ctypes.byref(self.L), n_seqs))

    def workspace(self, n_seqs: int) -> torch.Tensor:
        need = self.workspace_bytes(n_seqs)
        if self._ws is None or self._ws.numel() < need:
            self._ws = torch.empty(need, device=self.device, dtype=torch.uint8)
        return self._ws

    def step(self, x, y, conv_state, state, workspace=None):
        """One decode step; a float16 `state` takes the fp16-state entry."""
        n_seqs = x.shape[0]
        ws = workspace if workspace is not None else self.workspace(n_seqs)
        name = "li_launch_deltanet_layer_decode_f16state" if state.dtype == torch.float16 else \
            "li_launch_deltanet_layer_decode"
        check(getattr(_lib.load(), name)(
            ctypes.byref(self.L), _p(x), _p(y), _p(conv_state), _p(state), n_seqs, _p(ws), ws.numel(),
            _stream()), name)
        return y


class AttnLayerDecode:
    """One gated attention layer's device weights plus a workspace, stepping
    B sequences one token at a time through li_launch_attn_layer_decode
    against caller-owned fp16 KV caches [B, max_ctx, Hkv, D]."""

    def __init__(self, *, hidden, n_q_heads, n_kv_heads, head_dim, w_in, w_out, rope_dim=64,
                 rope_theta=1e7, in_norm_w=None, q_norm_w=None, k_norm_w=None, w_in_type=LI_WTYPE_Q4_K,
                 w_out_type=LI_WTYPE_Q4_K, in_norm_eps=1e-6, qk_norm_eps=1e-6):
        self.keep = [w_in, w_out, in_norm_w, q_norm_w, k_norm_w]
        self.L = AttnLayer(
            hidden=hidden, n_q_heads=n_q_heads, n_kv_heads=n_kv_heads, head_dim=head_dim, rope_dim=rope_dim,
            w_in_type=w_in_type, w_out_type=w_out_type, rope_theta=rope_theta, in_norm_eps=in_norm_eps,
            qk_norm_eps=qk_norm_eps, in_norm_w=_p(in_norm_w), w_in=_p(w_in), q_norm_w=_p(q_norm_w),
            k_norm_w=_p(k_norm_w), w_out=_p(w_out))
        self.device = w_in.device
        self._ws = None

    def workspace_bytes(self, n_seqs: int, max_ctx: int) -> int:
        return int(_lib.load().li_attn_layer_workspace_size(ctypes.byref(self.L), n_seqs, max_ctx))

    def workspace(self, n_seqs: int, max_ctx: int) -> torch.Tensor:
        need = self.workspace_bytes(n_seqs, max_ctx)
        if self._ws is None or self._ws.numel() < need:
            self._ws = torch.empty(need, device=self.device, dtype=torch.uint8)
        return self._ws

    def step(self, x, y, k_cache, v_cache, pos, workspace=None):
        """One decode step: the new token of sequence s goes to slot pos[s]
        (an int32 device tensor) of the caches."""
        n_seqs, max_ctx = x.shape[0], k_cache.shape[1]
        ws = workspace if workspace is not None else self.workspace(n_seqs, max_ctx)
        check(_lib.load().li_launch_attn_layer_decode(
            ctypes.byref(self.L), _p(x), _p(y), _p(k_cache), _p(v_cache), _p(pos), n_seqs, max_ctx, _p(ws),
            ws.numel(), _stream()), "li_launch_attn_layer_decode")
        return y

    def step_kv(self, x, y, cache: "KVCache", pos, rope: "Rope | None" = None, decay: float = 1.0, workspace=None):
        """One decode step on a managed cache: the new token of sequence s, at
        position pos[s] (int32), goes to slot cache.len[s] - 1; rope defaults
        to the layer's own parameters."""
        _on(cache.index, x, y, pos, workspace, rope.keep if rope is not None else None, *self.keep)
        if x.shape != (cache.n_seqs, self.L.hidden) or y.shape != x.shape or x.dtype != y.dtype or \
                x.dtype != torch.float32:
            raise ValueError(f"x, y: expected fp32 [{cache.n_seqs}, {self.L.hidden}]")
        if cache.n_seqs == 0:
            return y
        lib, L = _lib.load(), self.L
        ws = workspace if workspace is not None else cache._workspace(
            ("layer", L.hidden, L.n_q_heads, L.w_in_type, L.w_out_type), lambda: int(lib.li_attn_layer_kv_workspace_size(ctypes.byref(self.L), cache.ref)))
        check(lib.li_launch_attn_layer_decode_kv(
            ctypes.byref(self.L), rope.ref if rope is not None else None, cache.ref, _p(x), _p(y),
            _index(pos, cache.n_seqs, "pos"), decay, ws.data_ptr(), ws.numel(), _stream()),
            "li_launch_attn_layer_decode_kv")
        return y


# --------------------------------------------------------------------------
# Rotary positions and the managed KV cache
# --------------------------------------------------------------------------
_DTYPES = {torch.float32: LI_DTYPE_F32, torch.float16: LI_DTYPE_F16, torch.bfloat16: LI_DTYPE_BF16}
_ROPE_LAYOUTS = {"interleaved": LI_ROPE_INTERLEAVED, "half": LI_ROPE_HALF}


def _on(index: int, *tensors) -> None:
    """The tensors lie on cuda:index, and it is the current device (the
    library launches on the current device's stream)."""
    if index < 0:
        raise ValueError("LeanInfer kernels take CUDA tensors")
    if index != torch.cuda.current_device():
        raise ValueError(f"tensors on cuda:{index}, but cuda:{torch.cuda.current_device()} is the current device")
    for t in tensors:
        if t is not None and t.get_device() != index:
            raise ValueError("LeanInfer kernels take CUDA tensors of one device")


def _heads(t: torch.Tensor, n: int, heads: int, dim: int, dtype, what: str) -> int:
    """Checks [n, heads, dim] with each token's heads contiguous and any token
    stride; returns that stride."""
    if t.shape != (n, heads, dim):
        raise ValueError(f"{what}: expected [{n}, {heads}, {dim}], got {tuple(t.shape)}")
    token, head, one = t.stride()
    if one != 1 or (head != dim and heads > 1):
        raise ValueError(f"{what}: the heads of a token must be contiguous")
    if t.dtype is not dtype:
        raise ValueError(f"{what}: expected {dtype}, got {t.dtype}")
    return token


def _index(t: torch.Tensor | None, n: int, what: str) -> int | None:
    if t is None:
        return None
    if t.dtype is not torch.int32 or t.shape != (n,) or not t.is_contiguous():
        raise ValueError(f"{what}: expected a contiguous int32 tensor of {n} values")
    return t.data_ptr()


class Rope:
    """Rotary position parameters (li_rope): layout "half" or "interleaved",
    the first rope_dim dims of head_dim, position interpolation (freq_scale)
    and YaRN (ext_factor 1 with n_ctx_orig, beta_fast, beta_slow),
    freq_factors an fp32 device tensor of rope_dim / 2 divisors or None."""

    def __init__(self, *, head_dim: int, rope_dim: int | None = None, layout: str = "half", theta: float = 1e7,
                 freq_scale: float = 1.0, ext_factor: float = 0.0, attn_factor: float = 1.0, beta_fast: float = 32.0,
                 beta_slow: float = 1.0, n_ctx_orig: int = 0, freq_factors: torch.Tensor | None = None):
        rope_dim = head_dim if rope_dim is None else rope_dim
        if layout not in _ROPE_LAYOUTS:
            raise ValueError(f"layout {layout!r}: expected one of {sorted(_ROPE_LAYOUTS)}")
        if freq_factors is not None and (freq_factors.dtype != torch.float32 or freq_factors.numel() != rope_dim // 2):
            raise ValueError(f"freq_factors: expected {rope_dim // 2} fp32 values")
        self.keep = freq_factors
        self.R = RopeParams(layout=_ROPE_LAYOUTS[layout], head_dim=head_dim, rope_dim=rope_dim, n_ctx_orig=n_ctx_orig,
                            theta=theta, freq_scale=freq_scale, ext_factor=ext_factor, attn_factor=attn_factor,
                            beta_fast=beta_fast, beta_slow=beta_slow, freq_factors=_p(freq_factors))
        self.head_dim = head_dim
        self.ref = ctypes.byref(self.R)


def rope(rope: Rope, x: torch.Tensor, pos: torch.Tensor, out: torch.Tensor | None = None, transpose: bool = False):
    """x [tokens, heads, head_dim] (fp32, fp16 or bf16; any token and head
    strides) rotated to the positions pos (int32 [tokens]); transpose: the
    transposed rotation (its gradient). out may be x."""
    n, heads, dim = x.shape
    if dim != rope.head_dim or x.stride(2) != 1:
        raise ValueError(f"x: expected [tokens, heads, {rope.head_dim}] with contiguous heads")
    if out is None:
        out = torch.empty(n, heads, dim, device=x.device, dtype=x.dtype)
    elif out.shape != x.shape or out.stride(2) != 1:
        raise ValueError("out: expected the shape of x with contiguous heads")
    if x.dtype not in _DTYPES:
        raise ValueError(f"x: {x.dtype} is not fp32, fp16 or bf16")
    if out.dtype != x.dtype:
        raise ValueError(f"out: expected {x.dtype}, got {out.dtype}")
    _on(x.get_device(), out, pos, rope.keep)
    if x.numel() == 0:
        return out
    xs, os = x.stride(), out.stride()
    check(_lib.load().li_launch_rope(rope.ref, _DTYPES[x.dtype], x.data_ptr(), out.data_ptr(), _index(pos, n, "pos"),
                                     n, heads, xs[0], xs[1], os[0], os[1], transpose, _stream()), "li_launch_rope")
    return out


class KVCache:
    """One attention layer's KV cache (li_kv_cache) over the caller's tensors:
    k, v fp16 [n_seqs, max_ctx, n_kv_heads, 128]; len int32 [n_seqs], the slots
    in use, which the caller advances before a step's append; an optional
    shared prefix fp16 [n_prefix, n_kv_heads, 128]; weight fp32 and slot_pos
    int32 [n_seqs, n_kv_heads, max_ctx] for the eviction. Workspaces are kept
    by the object, and captured graphs hold their addresses: calls and replays
    that overlap on the GPU need an object each, and the object has to live as
    long as the graphs."""

    def __init__(self, k, v, len, *, k_prefix=None, v_prefix=None, weight=None, slot_pos=None):
        n, ctx, heads, dim = k.shape
        self.device, self.index = k.device, k.get_device()
        if v.shape != k.shape:
            raise ValueError("k and v differ in shape")
        if (k_prefix is None) != (v_prefix is None):
            raise ValueError("k_prefix and v_prefix go together")
        p = 0 if k_prefix is None else k_prefix.shape[0]
        if p and (tuple(k_prefix.shape) != (p, heads, dim) or v_prefix.shape != k_prefix.shape):
            raise ValueError(f"prefix: expected [n_prefix, {heads}, {dim}]")
        for t, dt in ((weight, torch.float32), (slot_pos, torch.int32)):
            if t is not None and (tuple(t.shape) != (n, heads, ctx) or t.dtype != dt):
                raise ValueError(f"weight and slot_pos: expected fp32 and int32 [{n}, {heads}, {ctx}]")
        for t in (k, v, k_prefix, v_prefix):
            if t is not None and t.dtype != torch.float16:
                raise ValueError("the cache rows are fp16")
        self.keep = [k, v, len, k_prefix, v_prefix, weight, slot_pos]
        for t in self.keep:
            if t is not None and t.device != k.device:
                raise ValueError(f"tensors on {t.device} and {k.device}")
        self.n_seqs, self.max_ctx, self.n_kv_heads, self.head_dim = n, ctx, heads, dim
        self.C = KvCache(n_seqs=n, max_ctx=ctx, n_kv_heads=heads, head_dim=dim, k=_p(k), v=_p(v),
                         len=_index(len, n, "len"), n_prefix=p, k_prefix=_p(k_prefix) if p else None,
                         v_prefix=_p(v_prefix) if p else None, weight=_p(weight), slot_pos=_p(slot_pos))
        self.ref = ctypes.byref(self.C)
        self._ws = {}

    def _workspace(self, key, size) -> torch.Tensor:
        ws = self._ws.get(key)
        if ws is None:
            ws = self._ws[key] = torch.empty(max(size(), 16), device=self.device, dtype=torch.uint8)
        return ws

    def append(self, k, v, pos, *, q=None, rope: Rope | None = None, seq=None, slot=None, q_out=None):
        """Appends k, v [tokens, n_kv_heads, 128] (k rotated to pos) at
        (seq[t], slot[t]), no two tokens at the same place; without seq, token
        t is sequence t's, without slot it goes to slot len - 1. Returns q
        rotated (q_out, which may be q), or None without q."""
        n, dt, dim = k.shape[0], k.dtype, self.head_dim
        if dt not in _DTYPES:
            raise ValueError(f"k: {dt} is not fp32, fp16 or bf16")
        ks, vs = _heads(k, n, self.n_kv_heads, dim, dt, "k"), _heads(v, n, self.n_kv_heads, dim, dt, "v")
        _on(self.index, k, v, q, q_out, pos, seq, slot, rope.keep if rope is not None else None)
        qp = op = None
        qs = os = hq = 0
        if q is not None:
            if q.dim() != 3:
                raise ValueError(f"q: expected [{n}, heads, {dim}]")
            hq = q.shape[1]
            qs = _heads(q, n, hq, dim, dt, "q")
            if q_out is None:
                q_out = torch.empty(n, hq, dim, device=self.device, dtype=dt)
            os = _heads(q_out, n, hq, dim, dt, "q_out")
            qp, op = q.data_ptr(), q_out.data_ptr()
        if n == 0:
            return q_out if q is not None else None
        check(_lib.load().li_launch_kv_append(
            self.ref, rope.ref if rope is not None else None, _DTYPES[dt], qp, qs, op, os, hq, k.data_ptr(), ks,
            v.data_ptr(), vs, _index(pos, n, "pos"), _index(seq, n, "seq"), _index(slot, n, "slot"), n, _stream()),
            "li_launch_kv_append")
        return q_out if q is not None else None

    def decode(self, q, *, scale: float | None = None, decay: float = 1.0, out=None, workspace=None):
        """Attention of q [n_seqs, n_q_heads, 128] (fp32) over the prefix and
        each sequence's first len slots; returns [n_seqs, n_q_heads, 128]. With
        weight in the cache, weight = decay * weight + this step's."""
        if q.dim() != 3:
            raise ValueError(f"q: expected [{self.n_seqs}, heads, {self.head_dim}]")
        hq = q.shape[1]
        qs = _heads(q, self.n_seqs, hq, self.head_dim, torch.float32, "q")
        if out is None:
            out = torch.empty(self.n_seqs, hq, self.head_dim, device=self.device, dtype=torch.float32)
        elif out.shape != q.shape or not out.is_contiguous() or out.dtype != torch.float32:
            raise ValueError("out: expected a contiguous fp32 tensor of q's shape")
        _on(self.index, q, out, workspace)
        if self.n_seqs == 0:
            return out
        lib = _lib.load()
        ws = workspace if workspace is not None else self._workspace(
            hq, lambda: int(lib.li_attn_kv_workspace_size(self.ref, hq)))
        check(lib.li_launch_attn_kv_decode(self.ref, q.data_ptr(), qs, hq,
                                           self.head_dim ** -0.5 if scale is None else scale, out.data_ptr(), decay,
                                           ws.data_ptr(), ws.numel(), _stream()), "li_launch_attn_kv_decode")
        return out

    def evict(self, pos, budget: int, *, n_sink: int = 0, n_recent: int = 0, workspace=None) -> None:
        """Shrinks every longer sequence to `budget` slots by weight (see
        li_launch_kv_evict); pos int32 [n_seqs], the newest token's position;
        n_sink counts own tokens, after the prefix."""
        _on(self.index, pos, workspace)
        if self.n_seqs == 0:
            return
        lib = _lib.load()
        # kept at the largest size that any budget needs (half of the slots): one for all of them
        ws = workspace if workspace is not None else self._workspace(
            "evict", lambda: int(lib.li_kv_evict_workspace_size(self.ref, self.max_ctx // 2)))
        check(lib.li_launch_kv_evict(self.ref, _index(pos, self.n_seqs, "pos"), budget, n_sink, n_recent,
                                     ws.data_ptr(), ws.numel(), _stream()), "li_launch_kv_evict")
