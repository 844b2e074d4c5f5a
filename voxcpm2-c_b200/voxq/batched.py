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

from . import BF16, F16, F32, RopeDesc, RopeTableDesc, LoraDesc, NormDesc, PagedAttnDesc, check, lib

_DTYPE = {torch.float32: F32, torch.float16: F16, torch.bfloat16: BF16}
ROPE_SCALING = {None: 0, "linear": 1, "ntk": 2, "yarn": 3, "long": 4}


def _code(t, what):
    c = _DTYPE.get(t.dtype)
    if c is None:
        raise ValueError(f"{what}: element type {t.dtype} is not float32, float16 or bfloat16")
    return c


def _need(ok, what):
    if not ok:
        raise ValueError(what)


def _ints(t, n, what, dtype=torch.int32):
    """Address of a contiguous device vector of n integers."""
    if t.dtype is not dtype or t.dim() != 1 or t.shape[0] != n or not t.is_cuda or (n > 1 and t.stride(0) != 1):
        raise ValueError(f"{what}: a contiguous CUDA vector of {n} {dtype} is needed")
    return t.data_ptr()


class _On:
    """The stream of a call: its handle, and allocation that belongs to it."""

    __slots__ = ("handle", "stream")

    def __init__(self, stream):
        if stream is None:
            self.handle, self.stream = torch.cuda.current_stream().cuda_stream, None
        elif hasattr(stream, "cuda_stream"):
            self.handle, self.stream = stream.cuda_stream, stream
        else:
            self.handle, self.stream = int(stream), torch.cuda.ExternalStream(int(stream))

    def empty(self, shape, dtype, device):
        if self.stream is None:
            return torch.empty(shape, dtype=dtype, device=device)
        with torch.cuda.stream(self.stream):
            return torch.empty(shape, dtype=dtype, device=device)


def rope_freqs(n_pos: int, rot_dim: int, theta: float = 10000.0, scaling: Optional[str] = None, factor: float = 1.0,
               original_len: int = 0, beta_fast: float = 32.0, beta_slow: float = 1.0, attn_factor: float = 1.0,
               long_factors: Optional[Sequence[float]] = None, device="cuda", stream=None):
    """cos and sin per position and pair, [n_pos, rot_dim / 2, 2] fp32 (voxq_rope_freqs; the engine's freqs_cis,
    src/tensor.c:883-950).  scaling: None, "linear", "ntk", "yarn" or "long" (a factor per pair)."""
    _need(scaling in ROPE_SCALING, f"unknown scaling {scaling!r}")
    _need(n_pos >= 0 and rot_dim >= 0 and rot_dim % 2 == 0, "n_pos >= 0 and an even rot_dim are needed")
    _need(scaling != "long" or (long_factors is not None and len(long_factors) == rot_dim // 2),
          "long scaling needs rot_dim / 2 factors")
    on = _On(stream)
    out = on.empty((n_pos, rot_dim // 2, 2), torch.float32, device)
    lf = (C.c_double * len(long_factors))(*long_factors) if scaling == "long" else None
    d = RopeTableDesc(n_pos, rot_dim, ROPE_SCALING[scaling], theta, factor, beta_fast, beta_slow, attn_factor,
                      original_len, C.cast(lf, C.c_void_p) if lf is not None else None, out.data_ptr())
    check(lib().voxq_rope_freqs(C.byref(d), on.handle), "voxq_rope_freqs")
    return out


def _rows3(t, what):
    """[tokens, heads, head_dim] with a contiguous last dimension, on the GPU."""
    if t.dim() != 3 or not t.is_cuda or (t.shape[2] > 1 and t.stride(2) != 1):
        raise ValueError(f"{what}: [tokens, heads, head_dim] on the GPU with a contiguous last dimension is needed")
    return t


def _caches(k, v, head_dim):
    if k.dim() != 4 or k.shape != v.shape or k.dtype is not v.dtype or k.stride() != v.stride() or not k.is_cuda \
            or not v.is_cuda or k.stride(3) != 1 or k.shape[3] != head_dim:
        raise ValueError("caches: two [pages, page_size, kv_heads, head_dim] CUDA tensors of one type and layout, "
                         "contiguous along head_dim, are needed")
    return k.stride()


def rope_append(q, k, v, freqs, positions, slots, cache_k, cache_v, q_out=None, interleaved: bool = False, stream=None):
    """Rotates q and k and writes k and v into a paged cache in one pass (voxq_rope_append); returns the rotated
    queries in the caches' type.  q [T, heads, D]; k, v [T, kv_heads, D]; freqs [n_pos, rot / 2, 2] (None: no
    rotation); positions int32 [T]; slots int64 [T], page * page_size + offset, -1 for padding rows."""
    T, H, D = _rows3(q, "q").shape
    KVH = _rows3(k, "k").shape[1]
    _need(k.shape == (T, KVH, D) and _rows3(v, "v").shape == (T, KVH, D), "q, k and v disagree in tokens or head_dim")
    _need(k.dtype is q.dtype and v.dtype is q.dtype, "q, k and v are of one type")
    sp, sr, sh, _ = _caches(cache_k, cache_v, D)
    _need(cache_k.shape[2] == KVH, "the caches' kv_heads differ from k's")
    on = _On(stream)
    if q_out is None:
        q_out = on.empty((T, H, D), cache_k.dtype, q.device)
    else:
        _need(_rows3(q_out, "q_out").shape == q.shape and q_out.dtype is cache_k.dtype, "q_out: q's shape, the caches' type")
    n_pos = rot = f = 0
    if freqs is not None:
        _need(freqs.dim() == 3 and freqs.shape[2] == 2 and freqs.dtype is torch.float32 and freqs.is_cuda
              and freqs.is_contiguous(), "freqs: contiguous fp32 [n_pos, rot / 2, 2] on the GPU")
        n_pos, rot, f = freqs.shape[0], 2 * freqs.shape[1], freqs.data_ptr()
    qs, ks, vs, os_ = q.stride(), k.stride(), v.stride(), q_out.stride()
    d = RopeDesc(q.data_ptr(), k.data_ptr(), v.data_ptr(), qs[0], qs[1], ks[0], ks[1], vs[0], vs[1], q_out.data_ptr(),
                 os_[0], os_[1], cache_k.data_ptr(), cache_v.data_ptr(), sp, sr, sh, f,
                 _ints(positions, T, "positions") if rot else 0, _ints(slots, T, "slots", torch.int64), T, H, KVH, D, rot,
                 interleaved, n_pos, cache_k.shape[0], cache_k.shape[1], _code(q, "q"), _code(cache_k, "cache_k"))
    check(lib().voxq_rope_append(C.byref(d), on.handle), "voxq_rope_append")
    return q_out


def paged_attention(q, cache_k, cache_v, block_table, cu_q, kv_len, max_q: int, max_kv: int, causal: bool = True,
                    scale: float = 0.0, out=None, out_dtype=None, stream=None):
    """Attention of each sequence's new tokens over its pages (voxq_paged_attention).  q [T, heads, D]; caches
    [pages, page_size, kv_heads, D] of q's type; block_table int32 [batch, width]; cu_q int32 [batch + 1]; kv_len
    int32 [batch], the new tokens included; max_q, max_kv: upper bounds of both.  scale 0: 1 / sqrt(D).  out_dtype:
    q's type (default) or torch.float32."""
    T, H, D = _rows3(q, "q").shape
    sp, sr, sh, _ = _caches(cache_k, cache_v, D)
    pages, page_size, KVH, _ = cache_k.shape
    _need(cache_k.dtype is q.dtype, "q and the caches are of one type")
    B = kv_len.shape[0]
    _need(block_table.dim() == 2 and block_table.shape[0] == B and block_table.dtype is torch.int32 and block_table.is_cuda
          and block_table.stride(1) == 1, "block_table: int32 [batch, width] on the GPU")
    _need(max_kv <= block_table.shape[1] * page_size, "max_kv is more than the block table's pages hold")
    on = _On(stream)
    if out is None:
        out = on.empty((T, H, D), out_dtype or q.dtype, q.device)
    else:
        _need(_rows3(out, "out").shape == q.shape, "out: q's shape")
    qs, os_ = q.stride(), out.stride()
    L = lib()
    d = PagedAttnDesc(q.data_ptr(), qs[0], qs[1], out.data_ptr(), os_[0], os_[1], cache_k.data_ptr(), cache_v.data_ptr(),
                      sp, sr, sh, block_table.data_ptr(), block_table.stride(0), _ints(cu_q, B + 1, "cu_q"),
                      _ints(kv_len, B, "kv_len"), B, H, KVH, D, pages, page_size, T, max_q, max_kv, _code(q, "q"),
                      _code(out, "out"), causal, scale, 0, 0)
    need = L.voxq_paged_attention_workspace(C.byref(d))
    if need:
        ws = on.empty((need,), torch.uint8, q.device)
        d.workspace, d.workspace_bytes = ws.data_ptr(), need
    check(L.voxq_paged_attention(C.byref(d), on.handle), "voxq_paged_attention")
    return out


def lora(x, a, b, cu, adapter, scale, base=None, out=None, ranks=None, stream=None):
    """out = base + scale[w] (x A[w]^T) B[w]^T for the rows of each request, w its adapter (voxq_lora_forward).
    x [rows, K]; a [adapters, rank, K]; b [adapters, N, rank]; cu int32 [batch + 1]; adapter int32 [batch], -1 for
    none; scale fp32 [adapters]; ranks int32 [adapters] or None; base [rows, N] or None; out may be base."""
    _need(x.dim() == 2 and x.is_cuda and (x.shape[1] <= 1 or x.stride(1) == 1), "x: [rows, K] on the GPU, contiguous along K")
    M, K = x.shape
    _need(a.dim() == 3 and b.dim() == 3 and a.is_contiguous() and b.is_contiguous() and a.is_cuda and b.is_cuda
          and a.dtype is b.dtype, "a, b: contiguous CUDA tensors of one type")
    nA, R, Ka = a.shape
    N = b.shape[1]
    _need(Ka == K and b.shape[0] == nA and b.shape[2] == R, "a is [adapters, rank, K] and b [adapters, N, rank]")
    _need(scale.dtype is torch.float32 and scale.is_cuda and scale.shape == (nA,) and scale.is_contiguous(),
          "scale: fp32 [adapters] on the GPU")
    B = adapter.shape[0]
    on = _On(stream)
    if out is None:
        out = on.empty((M, N), x.dtype, x.device)
    for t, what in ((base, "base"), (out, "out")):
        if t is not None:
            _need(t.shape == (M, N) and t.dtype is x.dtype and t.is_cuda and (N <= 1 or t.stride(1) == 1),
                  f"{what}: [rows, N] of x's type on the GPU")
    d = LoraDesc(x.data_ptr(), x.stride(0), 0 if base is None else base.data_ptr(), 0 if base is None else base.stride(0),
                 out.data_ptr(), out.stride(0), a.data_ptr(), b.data_ptr(), _ints(cu, B + 1, "cu"), _ints(adapter, B, "adapter"),
                 0 if ranks is None else _ints(ranks, nA, "ranks"), scale.data_ptr(), M, B, K, N, R, nA, _code(x, "x"), _code(a, "a"))
    check(lib().voxq_lora_forward(C.byref(d), on.handle), "voxq_lora_forward")
    return out


def norm_residual(y, x, w_pre=None, w_post=None, gate=None, gate_index=None, alpha: float = 1.0, eps: float = 1e-5,
                  h_out=None, n_out=None, stream=None):
    """(h, n) with h = x + alpha * gate * (RMSNorm(y) w_post, or y) and n = RMSNorm(h) w_pre (voxq_norm_residual;
    n is None without w_pre).  y, x [rows, D]; norm weights fp32 [D]; gate [gate_rows, D], its row gate_index[m]
    (int32 [rows]) for row m, or one gate row for all, or one per row."""
    _need(y.dim() == 2 and y.shape == x.shape and y.dtype is x.dtype and y.is_cuda and x.is_cuda
          and (y.shape[1] <= 1 or (y.stride(1) == 1 and x.stride(1) == 1)), "y, x: [rows, D] of one type on the GPU")
    M, D = y.shape
    for w, what in ((w_pre, "w_pre"), (w_post, "w_post")):
        if w is not None:
            _need(w.dtype is torch.float32 and w.is_cuda and w.shape == (D,) and w.is_contiguous(), f"{what}: fp32 [D] on the GPU")
    gr, g, ldg, gi = 0, 0, 0, 0
    if gate is not None:
        _need(gate.dim() == 2 and gate.shape[1] == D and gate.dtype is y.dtype and gate.is_cuda
              and (D <= 1 or gate.stride(1) == 1), "gate: [gate_rows, D] of y's type on the GPU")
        gr, g, ldg = gate.shape[0], gate.data_ptr(), gate.stride(0)
        gi = 0 if gate_index is None else _ints(gate_index, M, "gate_index")
    on = _On(stream)
    if h_out is None:
        h_out = on.empty((M, D), y.dtype, y.device)
    if n_out is None and w_pre is not None:
        n_out = on.empty((M, D), y.dtype, y.device)
    _need(w_pre is not None or n_out is None, "n_out needs w_pre")
    for t, what in ((h_out, "h_out"), (n_out, "n_out")):
        if t is not None:
            _need(t.shape == (M, D) and t.dtype is y.dtype and t.is_cuda and (D <= 1 or t.stride(1) == 1),
                  f"{what}: [rows, D] of y's type on the GPU")
    d = NormDesc(y.data_ptr(), x.data_ptr(), g, y.stride(0), x.stride(0), ldg, 0 if w_post is None else w_post.data_ptr(),
                 0 if w_pre is None else w_pre.data_ptr(), gi, h_out.data_ptr(), 0 if n_out is None else n_out.data_ptr(),
                 h_out.stride(0), 0 if n_out is None else n_out.stride(0), M, D, gr, _code(y, "y"), alpha, eps)
    check(lib().voxq_norm_residual(C.byref(d), on.handle), "voxq_norm_residual")
    return h_out, n_out
