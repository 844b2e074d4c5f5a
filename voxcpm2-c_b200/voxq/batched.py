"""A decoder step over many utterances: the operators of include/voxq.h's ragged batch, on torch CUDA tensors.

The tokens of all sequences are concatenated; sequence s owns rows cu[s] .. cu[s+1] - 1.  The reference runs one
sequence at a time (src/model.c:653).  Every function launches on `stream` (a torch stream or a raw handle;
default: the current one), allocates its outputs and workspaces for that stream, and raises ``VoxqError`` with the
library's code, or ``ValueError`` for a tensor whose type, shape or device does not fit.
"""
from __future__ import annotations

import ctypes as C
from typing import Optional, Sequence

import torch

from . import RopeTableDesc, VoxqError, _torch, check, lib

ROPE_SCALING = {None: 0, "linear": 1, "ntk": 2, "yarn": 3, "long": 4}
_torch.bind(*(C.cast(lib()[f], C.c_void_p).value for f in (
    "voxq_rope_append", "voxq_paged_attention", "voxq_paged_attention_workspace", "voxq_lora_forward",
    "voxq_norm_residual")), VoxqError)


def _need(ok, what):
    if not ok:
        raise ValueError(what)


def _on(stream, device):
    """Makes `stream` the current one of `device`: outputs and workspaces that a call makes then belong to it, and are
    not handed out again while the call uses them."""
    if not hasattr(stream, "cuda_stream"):
        stream = torch.cuda.ExternalStream(int(stream), device=device)
    _need(stream.device == device, f"a stream of {stream.device} for tensors on {device}")
    return torch.cuda.stream(stream)


def _device(t):
    """Where a call runs: its first tensor's GPU."""
    _need(isinstance(t, torch.Tensor) and t.is_cuda, "a CUDA tensor is needed")
    return t.device


def rope_freqs(n_pos: int, rot_dim: int, theta: float = 10000.0, scaling: Optional[str] = None, factor: float = 1.0,
               original_len: int = 0, beta_fast: float = 32.0, beta_slow: float = 1.0, attn_factor: float = 1.0,
               long_factors: Optional[Sequence[float]] = None, device="cuda", stream=None):
    """cos and sin per position and pair, [n_pos, rot_dim / 2, 2] fp32 (voxq_rope_freqs; the engine's freqs_cis,
    src/tensor.c:883-950).  scaling: None, "linear", "ntk", "yarn" or "long" (a factor per pair)."""
    _need(scaling in ROPE_SCALING, f"unknown scaling {scaling!r}")
    _need(n_pos >= 0 and rot_dim >= 0 and rot_dim % 2 == 0, "n_pos >= 0 and an even rot_dim are needed")
    _need(scaling != "long" or (long_factors is not None and len(long_factors) == rot_dim // 2),
          "long scaling needs rot_dim / 2 factors")
    if stream is not None:
        device = torch.empty(0, device=device).device
        with _on(stream, device):
            return rope_freqs(n_pos, rot_dim, theta, scaling, factor, original_len, beta_fast, beta_slow, attn_factor,
                              long_factors, device)
    out = torch.empty((n_pos, rot_dim // 2, 2), dtype=torch.float32, device=device)
    if out.numel() == 0:
        return out
    _need(out.is_cuda, "device: a GPU is needed")
    lf = (C.c_double * len(long_factors))(*long_factors) if scaling == "long" else None
    d = RopeTableDesc(n_pos, rot_dim, ROPE_SCALING[scaling], theta, factor, beta_fast, beta_slow, attn_factor,
                      original_len, C.cast(lf, C.c_void_p) if lf is not None else None, out.data_ptr())
    with torch.cuda.device(out.device):
        check(lib().voxq_rope_freqs(C.byref(d), torch.cuda.current_stream().cuda_stream), "voxq_rope_freqs")
    return out


# The calls below hand their arguments to csrc/voxq_torch.cpp, which checks the tensors, makes the outputs and calls the
# library: the same from Python took 8 us a call where a small step's kernel takes 2 to 3.

def rope_append(q, k, v, freqs, positions, slots, cache_k, cache_v, q_out=None, interleaved: bool = False, stream=None):
    """Rotates q and k and writes k and v into a paged cache in one pass (voxq_rope_append); returns the rotated
    queries in the caches' type.  q [T, heads, D]; k, v [T, kv_heads, D]; freqs [n_pos, rot / 2, 2] (None: no
    rotation); positions int32 [T]; slots int64 [T], page * page_size + offset, -1 for padding rows."""
    if stream is not None:
        with _on(stream, _device(q)):
            return rope_append(q, k, v, freqs, positions, slots, cache_k, cache_v, q_out, interleaved)
    return _torch.rope_append(q, k, v, freqs, positions, slots, cache_k, cache_v, q_out, interleaved)


def paged_attention(q, cache_k, cache_v, block_table, cu_q, kv_len, max_q: int, max_kv: int, causal: bool = True,
                    scale: float = 0.0, out=None, out_dtype=None, stream=None):
    """Attention of each sequence's new tokens over its pages (voxq_paged_attention).  q [T, heads, D]; caches
    [pages, page_size, kv_heads, D] of q's type; block_table int32 [batch, width]; cu_q int32 [batch + 1]; kv_len
    int32 [batch], the new tokens included; max_q, max_kv: upper bounds of both.  scale 0: 1 / sqrt(D).  out_dtype:
    q's type (default) or torch.float32."""
    if stream is not None:
        with _on(stream, _device(q)):
            return paged_attention(q, cache_k, cache_v, block_table, cu_q, kv_len, max_q, max_kv, causal, scale, out, out_dtype)
    _need(out is None or out_dtype is None or out.dtype == out_dtype, "out and out_dtype differ")
    if out is None and out_dtype is not None:
        out = torch.empty(q.shape, dtype=out_dtype, device=q.device)
    return _torch.paged_attention(q, cache_k, cache_v, block_table, cu_q, kv_len, max_q, max_kv, causal, scale, out)


def lora(x, a, b, cu, adapter, scale, base=None, out=None, ranks=None, stream=None):
    """out = base + scale[w] (x A[w]^T) B[w]^T for the rows of each request, w its adapter (voxq_lora_forward).
    x [rows, K]; a [adapters, rank, K]; b [adapters, N, rank]; cu int32 [batch + 1]; adapter int32 [batch], -1 for
    none; scale fp32 [adapters]; ranks int32 [adapters] or None; base [rows, N] or None; out may be base."""
    if stream is not None:
        with _on(stream, _device(x)):
            return lora(x, a, b, cu, adapter, scale, base, out, ranks)
    return _torch.lora(x, a, b, cu, adapter, scale, base, out, ranks)


def norm_residual(y, x, w_pre=None, w_post=None, gate=None, gate_index=None, alpha: float = 1.0, eps: float = 1e-5,
                  h_out=None, n_out=None, stream=None):
    """(h, n) with h = x + alpha * gate * (RMSNorm(y) w_post, or y) and n = RMSNorm(h) w_pre (voxq_norm_residual;
    n is None without w_pre).  y, x [rows, D]; norm weights fp32 [D]; gate [gate_rows, D], its row gate_index[m]
    (int32 [rows]) for row m, or one gate row for all, or one per row."""
    if stream is not None:
        with _on(stream, _device(y)):
            return norm_residual(y, x, w_pre, w_post, gate, gate_index, alpha, eps, h_out, n_out)
    return _torch.norm_residual(y, x, w_pre, w_post, gate, gate_index, alpha, eps, h_out, n_out)
