"""Plain 64-bit forms of the batched-step operators (host float64, loops over sequences and heads) and the error
bounds that the tests hold the kernels to.

Bounds, per element, from the arithmetic alone.  u is the unit roundoff of the output type (2^-24, 2^-11, 2^-8 for
fp32, fp16, bf16: half an ulp relative to the value's binade), e = 2^-24 that of the fp32 arithmetic:
  attention  u |o| + (2 u_p + 4 delta + L e + 8 e) sum_j p_j |v_j|: u_p = u of the 16-bit types (the softmax weights
             enter the second product in the operand type; numerator and sum), 0 for fp32; delta = (D + 4) e times
             the largest sum_d |q_d k_jd| scale (a score's error moves p by that much, numerator and sum, twice over
             for the running maximum); L keys summed in fp32
  rotation   u |y| + 4 e (|x0| + |x1|): two products and one sum
  adapters   u |out| + e |base| + (K + rank + 8) e scale sum |x| |A| |B| + 2^-16 scale sum_r |h_r| |B_r|: h enters
             the second product with at least 16 significant bits
  norms      u |n| + (D / 2 + 16) e |n|, and for h u |h| + ((D / 2 + 16) e) alpha |g z| + 4 e (|x| + alpha |g z|)
"""
from __future__ import annotations

import torch

U = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
E = 2.0 ** -24
# a 16-bit result below the type's normal range is rounded to a multiple of its smallest subnormal
TINY = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -24, torch.bfloat16: 2.0 ** -133}


def f8(t):
    return t.detach().cpu().double()


def assert_within(y, ref, bound, what=""):
    y = f8(y)
    assert y.shape == ref.shape, f"{what}: shape {tuple(y.shape)}, not {tuple(ref.shape)}"
    assert torch.isfinite(y).all(), f"{what}: {int((~torch.isfinite(y)).sum())} values are not finite"
    over = (y - ref).abs() - bound
    if (over > 0).any():
        i = tuple(int(x) for x in torch.unravel_index(over.argmax(), over.shape))
        raise AssertionError(f"{what}: {int((over > 0).sum())} of {over.numel()} beyond the bound; worst at {i}: "
                             f"{float(y[i])!r}, not {float(ref[i])!r}, bound {float(bound[i]):.3e}")


def attention(q, ck, cv, table, cu, kv_len, causal, scale, out_dtype=None):
    """(result, bound) of paged attention, in float64 on the host."""
    dt = q.dtype
    q, ck, cv, table, cu, kv_len = f8(q), f8(ck), f8(cv), table.cpu().long(), cu.tolist(), kv_len.tolist()
    T, H, D = q.shape
    page, KVH = ck.shape[1], ck.shape[2]
    out, bound = torch.zeros_like(q), torch.zeros_like(q)
    up = 0.0 if dt is torch.float32 else U[dt]
    uo = U[out_dtype or dt]
    for s, L in enumerate(kv_len):
        n = cu[s + 1] - cu[s]
        if n == 0 or L == 0:
            continue
        pos = torch.arange(L)
        at = table[s, pos // page] * page + pos % page
        k, v = ck.flatten(0, 1)[at], cv.flatten(0, 1)[at]
        seen = torch.ones(n, L, dtype=torch.bool)
        if causal:
            seen = pos[None] <= (L - n + torch.arange(n))[:, None]
        for h in range(H):
            qq, kk, vv = q[cu[s]:cu[s + 1], h], k[:, h * KVH // H], v[:, h * KVH // H]
            sc = (qq @ kk.T * scale).masked_fill(~seen, -torch.inf)
            p = torch.exp(sc - sc.amax(1, keepdim=True).clamp(min=-1e300))
            tot = p.sum(1, keepdim=True)
            p = torch.where(tot > 0, p / tot.clamp(min=1e-300), torch.zeros_like(p))
            o, ab = p @ vv, p @ vv.abs()
            delta = ((qq.abs() @ kk.abs().T) * scale * seen).amax(1, keepdim=True) * (D + 4) * E
            out[cu[s]:cu[s + 1], h] = o
            bound[cu[s]:cu[s + 1], h] = uo * o.abs() + (2 * up + 4 * delta + (L + 8) * E) * ab + TINY[out_dtype or dt]
    return out, bound


def rotate(x, freqs, pos, interleaved, dtype):
    """(result, bound) of the rotation of x [T, heads, D]."""
    x, fr = f8(x), f8(freqs)[pos.cpu().long()]
    half = fr.shape[1]
    i0 = torch.arange(half) * 2 if interleaved else torch.arange(half)
    i1 = i0 + 1 if interleaved else i0 + half
    c, s = fr[:, None, :, 0], fr[:, None, :, 1]
    y, b = x.clone(), torch.zeros_like(x)
    y[..., i0] = x[..., i0] * c - x[..., i1] * s
    y[..., i1] = x[..., i0] * s + x[..., i1] * c
    both = 4 * E * (x[..., i0].abs() + x[..., i1].abs()) * f8(freqs).abs().max()
    b[..., i0] = both
    b[..., i1] = both
    return y, b + U[dtype] * y.abs() + TINY[dtype]


def adapters(x, a, b, cu, who, scale, base, ranks):
    dt = x.dtype
    x, a, b, scale, cu, who = f8(x), f8(a), f8(b), f8(scale), cu.tolist(), who.tolist()
    nA, R, K = a.shape
    out = torch.zeros(x.shape[0], b.shape[1], dtype=torch.float64) if base is None else f8(base).clone()
    bound = E * out.abs()
    for s, w in enumerate(who):
        if not 0 <= w < nA or cu[s] == cu[s + 1]:
            continue
        r = R if ranks is None else int(ranks[w])
        rows = slice(cu[s], cu[s + 1])
        h = x[rows] @ a[w, :r].T
        mag = x[rows].abs() @ a[w, :r].abs().T
        out[rows] += scale[w] * (h @ b[w, :, :r].T)
        bound[rows] += scale[w].abs() * ((K + r + 8) * E * (mag @ b[w, :, :r].abs().T) +
                                         2.0 ** -16 * (h.abs() @ b[w, :, :r].abs().T))
    return out, bound + U[dt] * out.abs() + TINY[dt]


def norm_residual(y, x, w_pre, w_post, gate, gate_index, alpha, eps):
    """((h, bound), (n, bound) or None)."""
    dt = y.dtype
    z, x = f8(y), f8(x)
    D = z.shape[1]
    rel = (D / 2 + 16) * E
    rms = lambda t: t / torch.sqrt((t * t).mean(1, keepdim=True) + eps)  # noqa: E731
    if w_post is not None:
        z = rms(z) * f8(w_post)
    if gate is not None:
        g = f8(gate)
        z = z * (g[gate_index.cpu().long()] if gate_index is not None else g)
    h = x + alpha * z
    hb = rel * (alpha * z).abs() + 4 * E * (x.abs() + (alpha * z).abs())
    if w_pre is None:
        return (h, hb + U[dt] * h.abs() + TINY[dt]), None
    n = rms(h) * f8(w_pre)
    inv = 1.0 / torch.sqrt((h * h).mean(1, keepdim=True) + eps)
    # h's own error reaches n directly and through the row's norm
    nb = rel * n.abs() + (hb * inv + n.abs() / f8(w_pre).abs().clamp(min=1e-30) * (hb * h.abs()).mean(1, keepdim=True) * inv ** 2) \
        * f8(w_pre).abs()
    return (h, hb + U[dt] * h.abs() + TINY[dt]), (n, nb + U[dt] * n.abs() + TINY[dt])
