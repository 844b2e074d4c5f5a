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

from . import BF16, F16, F32, LoraDesc, NormDesc, PagedAttnDesc, RopeDesc, RopeTableDesc, check, lib

_DTYPE = {torch.float32: F32, torch.float16: F16, torch.bfloat16: BF16}
ROPE_SCALING = {None: 0, "linear": 1, "ntk": 2, "yarn": 3, "long": 4}
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or \
    (lambda device: torch.cuda.current_stream(device).cuda_stream)


def _entry(name, *more, res=C.c_int):
    """A library function that takes its descriptor as packed bytes."""
    f = lib()[name]
    f.argtypes, f.restype = [C.c_char_p, *more], res
    return f


_rope_append = _entry("voxq_rope_append", C.c_void_p)
_paged_attention = _entry("voxq_paged_attention", C.c_void_p)
_paged_workspace = _entry("voxq_paged_attention_workspace", res=C.c_size_t)
_lora_forward = _entry("voxq_lora_forward", C.c_void_p)
_norm_residual = _entry("voxq_norm_residual", C.c_void_p)
_pack_rope, _pack_attn, _pack_lora, _pack_norm = RopeDesc.pack, PagedAttnDesc.pack, LoraDesc.pack, NormDesc.pack
_like = torch.empty_like


def _need(ok, what):
    if not ok:
        raise ValueError(what)


def _vector(t, n, what, dtype=torch.int32):
    """Address of a contiguous device vector of n values."""
    if t.dtype is not dtype or t.numel() != n or not t.is_cuda or not t.is_contiguous():
        raise ValueError(f"{what}: a contiguous CUDA vector of {n} {dtype} is needed")
    return t.data_ptr()


def _handle(stream):
    """The raw handle of a torch stream, or a handle as it is."""
    return stream.cuda_stream if hasattr(stream, "cuda_stream") else int(stream)


def _empty(shape, dtype, device, stream):
    """Memory that belongs to the call's stream, so that it is not handed out again while the call uses it."""
    if stream is None:
        return torch.empty(shape, dtype=dtype, device=device)
    with torch.cuda.stream(stream if hasattr(stream, "cuda_stream") else torch.cuda.ExternalStream(int(stream))):
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
    out = _empty((n_pos, rot_dim // 2, 2), torch.float32, device, stream)
    if out.numel() == 0:
        return out
    lf = (C.c_double * len(long_factors))(*long_factors) if scaling == "long" else None
    d = RopeTableDesc(n_pos, rot_dim, ROPE_SCALING[scaling], theta, factor, beta_fast, beta_slow, attn_factor,
                      original_len, C.cast(lf, C.c_void_p) if lf is not None else None, out.data_ptr())
    check(lib().voxq_rope_freqs(C.byref(d), _raw_stream(out.get_device()) if stream is None else _handle(stream)), "voxq_rope_freqs")
    return out


# The calls below spend most of a small step's time in Python, so their checks are written out: one test per tensor,
# and the words for what is wrong only once something is.

def _refuse(t, dims, what):
    raise ValueError(f"{what}: a {dims}-dimensional CUDA tensor with a contiguous last dimension is needed")


def _caches(k, v, head_dim):
    shape, st = k.shape, k.stride()
    if len(st) != 4 or v.shape != shape or v.dtype is not k.dtype or v.stride() != st or not k.is_cuda \
            or not v.is_cuda or st[3] != 1 or shape[3] != head_dim:
        raise ValueError("caches: two [pages, page_size, kv_heads, head_dim] CUDA tensors of one type and layout, "
                         "contiguous along head_dim, are needed")
    return shape, st


def rope_append(q, k, v, freqs, positions, slots, cache_k, cache_v, q_out=None, interleaved: bool = False, stream=None):
    """Rotates q and k and writes k and v into a paged cache in one pass (voxq_rope_append); returns the rotated
    queries in the caches' type.  q [T, heads, D]; k, v [T, kv_heads, D]; freqs [n_pos, rot / 2, 2] (None: no
    rotation); positions int32 [T]; slots int64 [T], page * page_size + offset, -1 for padding rows."""
    qd, qs, kd, ks, vs, dt, ct = q.shape, q.stride(), k.shape, k.stride(), v.stride(), q.dtype, cache_k.dtype
    if len(qs) != 3 or qs[2] != 1 or not q.is_cuda:
        _refuse(q, 3, "q")
    if len(ks) != 3 or ks[2] != 1 or vs[-1] != 1 or not k.is_cuda or not v.is_cuda:
        _refuse(k, 3, "k, v")
    T, H, D = qd
    KVH = kd[1]
    if v.shape != kd or kd[0] != T or kd[2] != D or k.dtype is not dt or v.dtype is not dt:
        raise ValueError("q [T, heads, D] and k, v [T, kv_heads, D] of one type are needed")
    (pages, page_size, ckh, _), cs = _caches(cache_k, cache_v, D)
    if ckh != KVH:
        raise ValueError("the caches' kv_heads differ from k's")
    if q_out is None:
        if stream is None:
            q_out = _like(q) if ct is dt else _like(q, dtype=ct)
        else:
            q_out = _empty((T, H, D), ct, q.device, stream)
        os_ = q_out.stride()
    else:
        os_ = q_out.stride()
        if q_out.shape != qd or q_out.dtype is not ct or os_[2] != 1 or not q_out.is_cuda:
            raise ValueError("q_out: q's shape and the caches' type, contiguous along head_dim, on the GPU")
    n_pos = rot = f = pos = 0
    if freqs is not None:
        n_pos, pairs, two = freqs.shape
        if two != 2:
            raise ValueError("freqs: [n_pos, rot / 2, 2]")
        f, rot, pos = _vector(freqs, n_pos * pairs * 2, "freqs", torch.float32), 2 * pairs, _vector(positions, T, "positions")
    code = _rope_append(_pack_rope(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), qs[0], qs[1], ks[0], ks[1], vs[0], vs[1], q_out.data_ptr(), os_[0], os_[1],
        cache_k.data_ptr(), cache_v.data_ptr(), cs[0], cs[1], cs[2], f, pos, _vector(slots, T, "slots", torch.int64), T, H,
        KVH, D, rot, 1 if interleaved else 0, n_pos, pages, page_size, _DTYPE.get(dt, -1), _DTYPE.get(ct, -1)),
        _raw_stream(q.get_device()) if stream is None else _handle(stream))
    if code:
        check(code, "voxq_rope_append")
    return q_out


def paged_attention(q, cache_k, cache_v, block_table, cu_q, kv_len, max_q: int, max_kv: int, causal: bool = True,
                    scale: float = 0.0, out=None, out_dtype=None, stream=None):
    """Attention of each sequence's new tokens over its pages (voxq_paged_attention).  q [T, heads, D]; caches
    [pages, page_size, kv_heads, D] of q's type; block_table int32 [batch, width]; cu_q int32 [batch + 1]; kv_len
    int32 [batch], the new tokens included; max_q, max_kv: upper bounds of both.  scale 0: 1 / sqrt(D).  out_dtype:
    q's type (default) or torch.float32."""
    qd, qs, dt = q.shape, q.stride(), q.dtype
    if len(qs) != 3 or qs[2] != 1 or not q.is_cuda:
        _refuse(q, 3, "q")
    T, H, D = qd
    (pages, page_size, KVH, _), cs = _caches(cache_k, cache_v, D)
    B = kv_len.numel()
    bt, ts = block_table.shape, block_table.stride()
    if len(ts) != 2 or (ts[1] != 1 and bt[1] > 1) or not block_table.is_cuda or cache_k.dtype is not dt or bt[0] != B \
            or block_table.dtype is not torch.int32:
        raise ValueError("caches of q's type and an int32 block_table [batch, width] on the GPU are needed")
    if max_kv > bt[1] * page_size:
        raise ValueError("max_kv is more than the block table's pages hold")
    if out is None:
        out = _like(q) if stream is None and out_dtype is None else _empty(qd, out_dtype or dt, q.device, stream)
        os_ = out.stride()
    else:
        os_ = out.stride()
        if out.shape != qd or os_[2] != 1 or not out.is_cuda:
            raise ValueError("out: q's shape, contiguous along head_dim, on the GPU")
    code, ocode = _DTYPE.get(dt, -1), _DTYPE.get(out.dtype, -1)
    d = (q.data_ptr(), qs[0], qs[1], out.data_ptr(), os_[0], os_[1], cache_k.data_ptr(), cache_v.data_ptr(), cs[0], cs[1],
         cs[2], block_table.data_ptr(), ts[0], _vector(cu_q, B + 1, "cu_q"), _vector(kv_len, B, "kv_len"), B, H, KVH, D, pages,
         page_size, T, max_q, max_kv, code, ocode, 1 if causal else 0, scale)
    packed = _pack_attn(*d, 0, 0)
    need = _paged_workspace(packed)
    if need:
        ws = _empty((need,), torch.uint8, q.device, stream)
        packed = _pack_attn(*d, ws.data_ptr(), need)
    code = _paged_attention(packed, _raw_stream(q.get_device()) if stream is None else _handle(stream))
    if code:
        check(code, "voxq_paged_attention")
    return out


def lora(x, a, b, cu, adapter, scale, base=None, out=None, ranks=None, stream=None):
    """out = base + scale[w] (x A[w]^T) B[w]^T for the rows of each request, w its adapter (voxq_lora_forward).
    x [rows, K]; a [adapters, rank, K]; b [adapters, N, rank]; cu int32 [batch + 1]; adapter int32 [batch], -1 for
    none; scale fp32 [adapters]; ranks int32 [adapters] or None; base [rows, N] or None; out may be base."""
    xs, dt = x.stride(), x.dtype
    if len(xs) != 2 or xs[1] != 1 or not x.is_cuda:
        _refuse(x, 2, "x")
    M, K = x.shape
    nA, R, Ka = a.shape
    nB, N, Rb = b.shape
    if Ka != K or nB != nA or Rb != R or a.dtype is not b.dtype or not a.is_contiguous() or not b.is_contiguous() \
            or not a.is_cuda or not b.is_cuda:
        raise ValueError("contiguous CUDA a [adapters, rank, K] and b [adapters, N, rank] of one type are needed")
    B = adapter.numel()
    bp = bs = 0
    if base is not None:
        bp, (bs, last) = base.data_ptr(), base.stride()
        if base.shape != (M, N) or base.dtype is not dt or last != 1 or not base.is_cuda:
            raise ValueError("base: [rows, N] of x's type, contiguous along N, on the GPU")
    if out is None:
        out = _like(base) if stream is None and base is not None else _empty((M, N), dt, x.device, stream)
        os_ = out.stride()
    else:
        os_ = out.stride()
        if out.shape != (M, N) or out.dtype is not dt or os_[1] != 1 or not out.is_cuda:
            raise ValueError("out: [rows, N] of x's type, contiguous along N, on the GPU")
    code = _lora_forward(_pack_lora(
        x.data_ptr(), xs[0], bp, bs, out.data_ptr(), os_[0], a.data_ptr(), b.data_ptr(), _vector(cu, B + 1, "cu"),
        _vector(adapter, B, "adapter"), 0 if ranks is None else _vector(ranks, nA, "ranks"),
        _vector(scale, nA, "scale", torch.float32), M, B, K, N, R, nA, _DTYPE.get(dt, -1), _DTYPE.get(a.dtype, -1)),
        _raw_stream(x.get_device()) if stream is None else _handle(stream))
    if code:
        check(code, "voxq_lora_forward")
    return out


def norm_residual(y, x, w_pre=None, w_post=None, gate=None, gate_index=None, alpha: float = 1.0, eps: float = 1e-5,
                  h_out=None, n_out=None, stream=None):
    """(h, n) with h = x + alpha * gate * (RMSNorm(y) w_post, or y) and n = RMSNorm(h) w_pre (voxq_norm_residual;
    n is None without w_pre).  y, x [rows, D]; norm weights fp32 [D]; gate [gate_rows, D], its row gate_index[m]
    (int32 [rows]) for row m, or one gate row for all, or one per row."""
    yd, ys, xs, dt = y.shape, y.stride(), x.stride(), y.dtype
    if len(ys) != 2 or (ys[1] != 1 and yd[1] > 1) or not y.is_cuda:
        _refuse(y, 2, "y")
    M, D = yd
    if x.shape != yd or x.dtype is not dt or (xs[1] != 1 and D > 1) or not x.is_cuda:
        raise ValueError("y and x: [rows, D] of one type, contiguous along D, on the GPU")
    g = gr = ldg = gi = np_ = ldn = wp = 0
    if gate is not None:
        gr, gD = gate.shape
        ldg, last = gate.stride()
        if gD != D or gate.dtype is not dt or (last != 1 and D > 1) or not gate.is_cuda:
            raise ValueError("gate: [gate_rows, D] of y's type, contiguous along D, on the GPU")
        g = gate.data_ptr()
        if gate_index is not None:
            gi = _vector(gate_index, M, "gate_index")
    if h_out is None:
        h_out = _like(y) if stream is None else _empty(yd, dt, y.device, stream)
    if w_pre is not None:
        wp = _vector(w_pre, D, "w_pre", torch.float32)
        if n_out is None:
            n_out = _like(y) if stream is None else _empty(yd, dt, y.device, stream)
        np_, (ldn, last) = n_out.data_ptr(), n_out.stride()
        if n_out.shape != yd or n_out.dtype is not dt or (last != 1 and D > 1) or not n_out.is_cuda:
            raise ValueError("n_out: [rows, D] of y's type, contiguous along D, on the GPU")
    elif n_out is not None:
        raise ValueError("n_out needs w_pre")
    ldh, last = h_out.stride()
    if h_out.shape != yd or h_out.dtype is not dt or (last != 1 and D > 1) or not h_out.is_cuda:
        raise ValueError("h_out: [rows, D] of y's type, contiguous along D, on the GPU")
    code = _norm_residual(_pack_norm(
        y.data_ptr(), x.data_ptr(), g, ys[0], xs[0], ldg, 0 if w_post is None else _vector(w_post, D, "w_post", torch.float32),
        wp, gi, h_out.data_ptr(), np_, ldh, ldn, M, D, gr, _DTYPE.get(dt, -1), alpha, eps),
        _raw_stream(y.get_device()) if stream is None else _handle(stream))
    if code:
        check(code, "voxq_norm_residual")
    return h_out, n_out
