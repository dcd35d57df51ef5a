"""Fused decode-step ops around the INT8 GEMV (functional layer over the C ABI).

These merge the torch ops that the reference runs inside the HF decoder layer
around its attention patch (helm/runtime/kv_offload.py:241-271 and transformers'
Qwen3DecoderLayer / Qwen3MLP): RMSNorm into the following projection, the
residual add into the projection epilogue, SiLU(gate) * up into the gate/up
projection, and q/k-norm + RoPE + the paged KV write into one kernel.
"""
from __future__ import annotations

from typing import Optional, Union

import torch

from .. import _native
from . import gemv_split_bytes
from .attention import _check_places


def _check_fp16(*ts):
    for t in ts:
        if t is not None and t.dtype != torch.float16:
            raise RuntimeError(f"expected fp16 tensor, got {t.dtype}")


def rmsnorm(x: torch.Tensor, weight: torch.Tensor, eps: float,
            out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """fp16(w * fp16(x * rsqrt(mean(x^2) + eps))) over the last dim (Qwen3RMSNorm)."""
    _native.require_cuda(x, weight, what="rmsnorm")
    _check_fp16(x, weight)
    K = x.shape[-1]
    x2 = x.reshape(-1, K).contiguous()
    if out is None:
        out = torch.empty_like(x2)
    _native.call("helm_rmsnorm", x2.data_ptr(), weight.data_ptr(), float(eps), out.data_ptr(),
                 x2.shape[0], K, _native.stream_ptr(x.device))
    return out.view(x.shape)


def qk_norm_rope_cs(qkv: torch.Tensor, q_norm_w: Optional[torch.Tensor],
                    k_norm_w: Optional[torch.Tensor], eps: float, cos: torch.Tensor,
                    sin: torch.Tensor, n_heads: int, n_kv_heads: int, head_dim: int):
    """(q [B, Hq, D], k [B, Hkv, D]) of the fused projection output qkv
    [B, (Hq + 2 Hkv) * D]: per-head RMSNorm (when the norm weights are given),
    then RoPE with the model's fp16 cos / sin rows [B, D] (helm_qk_norm_rope_cs)."""
    _native.require_cuda(qkv, q_norm_w, k_norm_w, cos, sin, what="qk_norm_rope_cs")
    _check_fp16(qkv, q_norm_w, k_norm_w, cos, sin)
    B = qkv.shape[0]
    if qkv.shape[-1] != (n_heads + 2 * n_kv_heads) * head_dim or not qkv.is_contiguous():
        raise RuntimeError("qk_norm_rope_cs: qkv must be contiguous [B, (Hq + 2 Hkv) * D]")
    if cos.shape[0] != B or cos.shape[-1] != head_dim or cos.stride(-1) != 1 or sin.stride() != cos.stride():
        raise RuntimeError("qk_norm_rope_cs: cos / sin must be [B, D] rows with unit stride")
    q = torch.empty(B, n_heads, head_dim, dtype=torch.float16, device=qkv.device)
    k = torch.empty(B, n_kv_heads, head_dim, dtype=torch.float16, device=qkv.device)
    _native.call("helm_qk_norm_rope_cs", qkv.data_ptr(), _native.ptr(q_norm_w), _native.ptr(k_norm_w),
                 float(eps), cos.data_ptr(), sin.data_ptr(), cos.stride(0), q.data_ptr(), k.data_ptr(),
                 B, n_heads, n_kv_heads, head_dim, _native.stream_ptr(qkv.device))
    return q, k


def int8_gemv_fused(x: torch.Tensor, qweight: torch.Tensor, scale: torch.Tensor,
                    norm_weight: Optional[torch.Tensor] = None, eps: float = 1e-6,
                    bias: Optional[torch.Tensor] = None,
                    residual: Optional[torch.Tensor] = None,
                    out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """y = [residual +] linear_int8(rmsnorm(x) if norm_weight else x), M <= 16 tokens."""
    _native.require_cuda(x, qweight, scale, norm_weight, bias, residual, what="int8_gemv_fused")
    _check_fp16(x, scale, norm_weight, bias, residual)
    N, K = qweight.shape
    x2 = x.reshape(-1, K).contiguous()
    M = x2.shape[0]
    if out is None:
        out = torch.empty(M, N, dtype=torch.float16, device=x.device)
    y2 = out.view(M, N)
    res = None
    if residual is not None:
        r2 = residual.reshape(M, N)
        if r2.data_ptr() == y2.data_ptr() or (r2.stride(1) == 1 and r2.stride(0) == y2.stride(0)):
            res = r2.data_ptr()          # read in place (row stride ldy, may alias y)
        else:
            y2.copy_(r2)
            res = y2.data_ptr()
    if norm_weight is None:
        # no norm prologue: the workspace form (split K for long K at 3-16 tokens)
        ws_bytes = gemv_split_bytes(M, N, K)
        ws = torch.empty(ws_bytes, dtype=torch.uint8, device=x.device) if ws_bytes else None
        _native.call("helm_int8_gemv_ws", x2.data_ptr(), x2.stride(0), qweight.data_ptr(),
                     qweight.stride(0), scale.data_ptr(), _native.ptr(bias), res, y2.data_ptr(),
                     y2.stride(0), M, N, K, _native.ptr(ws), ws_bytes, _native.stream_ptr(x.device))
        return out
    _native.call("helm_int8_gemv_fused", x2.data_ptr(), x2.stride(0), _native.ptr(norm_weight),
                 float(eps), qweight.data_ptr(), qweight.stride(0), scale.data_ptr(),
                 _native.ptr(bias), res, y2.data_ptr(), y2.stride(0), M, N, K,
                 _native.stream_ptr(x.device))
    return out


def int8_gemv_swiglu(x: torch.Tensor, q_gate: torch.Tensor, s_gate: torch.Tensor,
                     q_up: torch.Tensor, s_up: torch.Tensor,
                     norm_weight: Optional[torch.Tensor] = None, eps: float = 1e-6,
                     out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """fp16(silu(gate(xn)) * up(xn)), xn = rmsnorm(x) if norm_weight else x."""
    _native.require_cuda(x, q_gate, s_gate, q_up, s_up, norm_weight, what="int8_gemv_swiglu")
    _check_fp16(x, s_gate, s_up, norm_weight)
    N, K = q_gate.shape
    if tuple(q_up.shape) != (N, K) or q_up.stride(0) != q_gate.stride(0):
        raise RuntimeError("int8_gemv_swiglu: gate and up weights must have the same shape/stride")
    x2 = x.reshape(-1, K).contiguous()
    M = x2.shape[0]
    if out is None:
        out = torch.empty(M, N, dtype=torch.float16, device=x.device)
    _native.call("helm_int8_gemv_swiglu", x2.data_ptr(), x2.stride(0), _native.ptr(norm_weight),
                 float(eps), q_gate.data_ptr(), s_gate.data_ptr(), q_up.data_ptr(),
                 s_up.data_ptr(), q_gate.stride(0), out.data_ptr(), out.stride(0), M, N, K,
                 _native.stream_ptr(x.device))
    return out


def rope_inv_freq(head_dim: int, theta: float, device=None) -> torch.Tensor:
    """inv_freq[i] = 1 / theta^(2i / head_dim) in fp32, computed as transformers'
    Qwen3RotaryEmbedding.compute_default_rope_parameters does."""
    return (1.0 / (theta ** (torch.arange(0, head_dim, 2, dtype=torch.int64).to(
        device=device, dtype=torch.float) / head_dim))).float()


def qk_norm_rope_append(qkv: torch.Tensor, q_norm_w: torch.Tensor, k_norm_w: torch.Tensor,
                        eps: float, positions: torch.Tensor, inv_freq: torch.Tensor,
                        q_out: torch.Tensor, pool, slots: torch.Tensor, offsets: torch.Tensor,
                        num_q_heads: int, num_kv_heads: int, head_dim: int,
                        page_size: int) -> torch.Tensor:
    """q/k RMSNorm + RoPE of the fused qkv [B, (Hq+2Hkv)*D]; writes k, v into the
    page slots of `pool` (an attention.PoolView) and the rotated q into q_out
    [B, Hq, D]."""
    _native.require_cuda(qkv, q_norm_w, k_norm_w, positions, inv_freq, q_out, pool.k, pool.v,
                         slots, offsets, what="qk_norm_rope_append")
    B = qkv.shape[0]
    _native.call("helm_qk_norm_rope_append", qkv.data_ptr(), q_norm_w.data_ptr(),
                 k_norm_w.data_ptr(), float(eps), positions.data_ptr(), inv_freq.data_ptr(),
                 q_out.data_ptr(), pool.c_ref(), slots.data_ptr(), offsets.data_ptr(), B,
                 num_q_heads, num_kv_heads, head_dim, page_size, _native.stream_ptr(qkv.device))
    return q_out


def qk_norm_rope_append_q8(qkv: torch.Tensor, q_norm_w: Optional[torch.Tensor],
                           k_norm_w: Optional[torch.Tensor], eps: float, positions: torch.Tensor,
                           inv_freq: torch.Tensor, q_out: Optional[torch.Tensor], pool, slots: torch.Tensor,
                           offsets: torch.Tensor, num_q_heads: int, num_kv_heads: int, head_dim: int,
                           page_size: Optional[int] = None) -> torch.Tensor:
    """qk_norm_rope_append into an 8-bit pool (an attention.Q8PoolView): q/k RMSNorm (when
    the norm weights are given) + RoPE of the fused qkv [B, (Hq+2Hkv)*D] in fp32, the angle
    in 64 bits; the rotated q rounded to fp16 once into q_out [B, Hq, D], k and v quantised
    into (slots[b], offsets[b]) with a scale per token and head, as kv_append_q8 does (tokens
    with a place outside the pool are not kept, and no two name one place)."""
    what = "qk_norm_rope_append_q8"
    index = _native.gpu_of(what, qkv, q_norm_w, k_norm_w, positions, inv_freq, q_out, pool.k, slots, offsets)
    _check_fp16(qkv, q_norm_w, k_norm_w, q_out)
    Hq, Hkv, D = num_q_heads, num_kv_heads, head_dim
    if qkv.dim() != 2 or qkv.shape[1] != (Hq + 2 * Hkv) * D or qkv.stride(1) != 1:
        raise RuntimeError(f"{what}: qkv must be [B, (Hq + 2 Hkv) * D] with unit stride")
    if Hkv != pool.num_kv_heads or D != pool.head_dim:
        raise RuntimeError(f"{what}: {Hkv} heads of {D} do not fit the pool's {pool.num_kv_heads} of {pool.head_dim}")
    P = pool._check_page_size(page_size, what)
    B, width = qkv.shape
    if positions.dtype != torch.int32 or positions.shape != (B,) or not positions.is_contiguous():
        raise RuntimeError(f"{what}: positions must be int32 [{B}], contiguous")
    _check_places(what, slots, offsets, B)
    if inv_freq.dtype != torch.float32 or inv_freq.shape != (D // 2,) or not inv_freq.is_contiguous():
        raise RuntimeError(f"{what}: inv_freq must be fp32 [{D // 2}], contiguous")
    if (q_norm_w is None) != (k_norm_w is None):
        raise RuntimeError(f"{what}: give both q / k norm weights or neither")
    for w in (q_norm_w, k_norm_w):
        if w is not None and (w.shape != (D,) or not w.is_contiguous()):
            raise RuntimeError(f"{what}: norm weights must be [D], contiguous")
    if q_out is None:
        q_out = qkv.new_empty((B, Hq, D))
    elif q_out.shape != (B, Hq, D) or not q_out.is_contiguous():
        raise RuntimeError(f"{what}: q_out must be [B, Hq, D], contiguous")
    if B == 0:
        return q_out
    stride = qkv.stride(0) if B > 1 else width
    if stride % 8 or stride < width or qkv.data_ptr() % 16:
        qkv, stride = qkv.clone(memory_format=torch.contiguous_format), width
    _native.call_on(index, "helm_qk_norm_rope_append_q8", qkv.data_ptr(), stride, _native.ptr(q_norm_w),
                    _native.ptr(k_norm_w), eps, positions.data_ptr(), inv_freq.data_ptr(), q_out.data_ptr(),
                    pool.c_ref(), slots.data_ptr(), offsets.data_ptr(), B, Hq, Hkv, D, P, _native.raw_stream(index))
    return q_out


def fp16_gemv_rmsnorm(x: torch.Tensor, norm_weight: torch.Tensor, eps: float,
                      weight: torch.Tensor, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """y = fp16(weight . rmsnorm(x)) for <= 16 tokens (final norm + lm_head)."""
    _native.require_cuda(x, norm_weight, weight, what="fp16_gemv_rmsnorm")
    _check_fp16(x, norm_weight, weight)
    N, K = weight.shape
    x2 = x.reshape(-1, K).contiguous()
    M = x2.shape[0]
    if out is None:
        out = torch.empty(M, N, dtype=torch.float16, device=x.device)
    _native.call("helm_fp16_gemv_rmsnorm", x2.data_ptr(), x2.stride(0), norm_weight.data_ptr(),
                 float(eps), weight.data_ptr(), weight.stride(0), out.data_ptr(), out.stride(0),
                 M, N, K, _native.stream_ptr(x.device))
    return out


def silu_mul(gate: torch.Tensor, up: torch.Tensor, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """fp16(fp16(silu(gate)) * up) elementwise (the fused SwiGLU epilogue's rounding)."""
    _native.require_cuda(gate, up, what="silu_mul")
    _check_fp16(gate)
    _check_fp16(up)
    if gate.shape != up.shape or not gate.is_contiguous() or not up.is_contiguous():
        raise RuntimeError("silu_mul: gate and up must be contiguous tensors of one shape")
    if out is None:
        out = torch.empty_like(gate)
    _native.call("helm_silu_mul", gate.data_ptr(), up.data_ptr(), out.data_ptr(), gate.numel(),
                 _native.stream_ptr(gate.device))
    return out


def argmax_workspace(M: int, device) -> torch.Tensor:
    """Workspace of helm_argmax_f16_ws for M rows (reusable across calls on one stream)."""
    n = int(_native.lib().helm_argmax_workspace_bytes(int(M)))
    return torch.empty(max(1, n // 4), dtype=torch.int32, device=device)


def argmax(x: torch.Tensor, out: Optional[torch.Tensor] = None,
           workspace: Optional[torch.Tensor] = None, single_workgroup: bool = False) -> torch.Tensor:
    """Index of the first maximum of each row of fp16 x [M, N] (torch.argmax(x, -1)):
    64 workgroups per row and a merge kernel (`workspace` from argmax_workspace,
    allocated here when not given), or with single_workgroup one workgroup per
    row and no workspace."""
    _native.require_cuda(x, what="argmax")
    _check_fp16(x)
    x2 = x.reshape(-1, x.shape[-1])
    if x2.stride(-1) != 1:
        x2 = x2.contiguous()
    M, N = x2.shape
    if out is None:
        out = torch.empty(M, dtype=torch.int64, device=x.device)
    stream = _native.stream_ptr(x.device)
    if single_workgroup:
        _native.call("helm_argmax_f16", x2.data_ptr(), x2.stride(0), M, N, out.data_ptr(), stream)
        return out
    if workspace is None:
        workspace = argmax_workspace(M, x.device)
    _native.require_cuda(workspace, what="argmax")
    _native.call("helm_argmax_f16_ws", x2.data_ptr(), x2.stride(0), M, N, out.data_ptr(),
                 workspace.data_ptr(), workspace.numel() * workspace.element_size(), stream)
    return out


def sample_workspace(M: int, N: int, device) -> torch.Tensor:
    """Workspace of helm_sample for M rows of N logits (reusable across calls on one
    stream; calls that overlap, or two graphs that may replay at once, need one each)."""
    return torch.empty(int(_native.lib().helm_sample_workspace_bytes(int(M), int(N))), dtype=torch.uint8,
                       device=device)


def sample(logits: torch.Tensor, u: torch.Tensor, temperature: Union[float, torch.Tensor] = 1.0,
           top_k: Union[int, torch.Tensor] = 0, top_p: Union[float, torch.Tensor] = 1.0,
           min_p: Union[float, torch.Tensor] = 0.0, out: Optional[torch.Tensor] = None,
           workspace: Optional[torch.Tensor] = None) -> torch.Tensor:
    """A token drawn from each row of fp16 logits [..., N], int64 [...], from the random
    numbers u [...] (fp32 in [0, 1)), beside `argmax` (helm_sample):

    weights exp((x - max) / temperature); of these the top_k largest (0: all; equal logits
    by index), of these the shortest prefix, by weight, that holds a share top_p, of these
    the ones of at least min_p times the largest; then, in index order, the token at which
    the summed weight passes u times the sum of all.  temperature 0 is `argmax`.  Each
    setting is a number, or a tensor with one per row (fp32, top_k int32).  At a temperature
    above 0 NaN logits are never drawn (`argmax` takes them as the largest) and a row with no
    logit above -inf gives 0.  N is at most 262144.  `workspace` from
    sample_workspace, allocated here when not given."""
    tensors = [x for x in (temperature, top_k, top_p, min_p) if torch.is_tensor(x)]
    index = _native.gpu_of("sample", logits, u, out, workspace, *tensors)
    _check_fp16(logits)
    if logits.dim() < 1 or logits.shape[-1] < 1:
        raise RuntimeError("sample: logits must be [..., N] with N >= 1")
    N = logits.shape[-1]
    x2 = logits if logits.dim() == 2 else logits.reshape(-1, N)
    M = x2.shape[0]
    if x2.stride(1) != 1 and N > 1 or M > 1 and x2.stride(0) < N:
        x2 = x2.contiguous()

    def rows(x, dtype, name):
        if x.dtype != dtype or x.numel() != M or not x.is_contiguous():
            raise RuntimeError(f"sample: {name} must be {dtype} with one number per row ({M}), contiguous")
        return x.data_ptr()

    def setting(x, dtype, name):
        return (rows(x, dtype, name), 0) if torch.is_tensor(x) else (None, x)
    up = rows(u, torch.float32, "u")
    tp, t = setting(temperature, torch.float32, "temperature")
    kp, k = setting(top_k, torch.int32, "top_k")
    pp, p = setting(top_p, torch.float32, "top_p")
    lp, lo = setting(min_p, torch.float32, "min_p")
    if not (t >= 0.0 and k >= 0 and p >= 0.0 and lo >= 0.0):
        raise RuntimeError("sample: temperature, top_k, top_p and min_p must not be negative")
    if out is None:
        out = logits.new_empty(logits.shape[:-1], dtype=torch.int64)
    elif out.dtype != torch.int64 or out.numel() != M or not out.is_contiguous():
        raise RuntimeError("sample: out must be int64 with one token per row, contiguous")
    if M == 0:
        return out
    if workspace is None:
        workspace = sample_workspace(M, N, logits.device)
    elif not workspace.is_contiguous():
        raise RuntimeError("sample: workspace must be contiguous")
    _native.call_on(index, "helm_sample", x2.data_ptr(), x2.stride(0) if M > 1 else N, M, N, up, tp, kp, pp, lp, t,
                    min(int(k), 2**31 - 1), p, lo, out.data_ptr(), workspace.data_ptr(), workspace.nbytes,
                    _native.raw_stream(index))
    return out
