"""Decoder blocks over many utterances at once: a paged KV cache and the transformer block on quantized weights.

The reference's transformer_block_forward (src/nn.c:579-700) takes one sequence with a contiguous cache;
``BatchedBlock`` computes the same function for every sequence of a ragged batch in one set of launches: the
norms (``norm_residual``), the quantized projections (``matmul_nt_q``) with a voice adapter per request beside them
(``lora``), rotary positions and the cache write (``rope_append``) and attention over the pages
(``paged_attention``).

    cache = PagedCache(layers=24, pages=4096, page_size=16, kv_heads=2, head_dim=128)
    step = cache.step([("anna", 37), ("ben", 1)], adapters={"ben": 3})   # 37 prompt tokens, one next token
    h, n = x, norm_residual(x, x, blocks[0].norm_attn, alpha=0.0)[1]
    for i, b in enumerate(blocks):
        h, n = b(h, n, step, cache, i, freqs, next_norm=blocks[i + 1].norm_attn if i + 1 < len(blocks) else out_norm)
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Dict, Hashable, List, Optional, Sequence, Tuple

import torch

from . import QWeight, matmul_nt_q
from .batched import lora, norm_residual, paged_attention, rope_append


@dataclass
class Step:
    """One step's ragged batch on the device (the operators' integer inputs) and its bounds on the host."""

    cu: torch.Tensor          # int32 [batch + 1]
    kv_len: torch.Tensor      # int32 [batch], this step's tokens included
    table: torch.Tensor       # int32 [batch, width]
    adapter: torch.Tensor     # int32 [batch], -1: none
    positions: torch.Tensor   # int32 [tokens]
    slots: torch.Tensor       # int64 [tokens]
    max_q: int
    max_kv: int
    tokens: int


class PagedCache:
    """Keys and values of all layers in pages of ``page_size`` positions, handed to sequences on demand.

    Page 0 belongs to no sequence (unused block-table entries point there).  ``step`` reserves the pages of a
    batch's new tokens and gives their places; ``release`` returns a finished sequence's pages."""

    def __init__(self, layers: int, pages: int, page_size: int, kv_heads: int, head_dim: int, dtype=torch.bfloat16,
                 device="cuda"):
        if pages < 2 or page_size < 1 or layers < 1:
            raise ValueError("at least 2 pages (page 0 is reserved), 1 layer and pages of 1 position are needed")
        shape = (layers, pages, page_size, kv_heads, head_dim)
        self.k, self.v = torch.empty(shape, dtype=dtype, device=device), torch.empty(shape, dtype=dtype, device=device)
        self.page_size, self.device = page_size, device
        self._free = list(range(pages - 1, 0, -1))
        self._pages: Dict[Hashable, List[int]] = {}
        self._len: Dict[Hashable, int] = {}

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def length(self, seq: Hashable) -> int:
        return self._len.get(seq, 0)

    def release(self, seq: Hashable) -> None:
        self._free.extend(reversed(self._pages.pop(seq, [])))
        self._len.pop(seq, None)

    def step(self, requests: Sequence[Tuple[Hashable, int]], adapters: Optional[Dict[Hashable, int]] = None) -> Step:
        """Appends ``n`` positions to each (sequence, n), new sequences included, and returns the batch.  MemoryError,
        with nothing changed, when the free pages do not suffice."""
        P = self.page_size
        if len({s for s, _ in requests}) != len(requests) or any(n < 0 for _, n in requests):
            raise ValueError("a step names each sequence once, with 0 or more new tokens")
        need = [max(0, -(-(self.length(s) + n) // P) - len(self._pages.get(s, []))) for s, n in requests]
        if sum(need) > len(self._free):
            raise MemoryError(f"{sum(need)} pages are needed and {len(self._free)} are free")
        cu, lens, rows, who, pos, slots = [0], [], [], [], [], []
        for (s, n), extra in zip(requests, need):
            own = self._pages.setdefault(s, [])
            own.extend(self._free.pop() for _ in range(extra))
            past = self.length(s)
            self._len[s] = past + n
            cu.append(cu[-1] + n)
            lens.append(past + n)
            rows.append(own)
            who.append((adapters or {}).get(s, -1))
            pos.extend(range(past, past + n))
            slots.extend(own[j // P] * P + j % P for j in range(past, past + n))
        width = max([len(r) for r in rows] + [1])
        i32 = lambda v: torch.tensor(v, dtype=torch.int32).to(self.device)  # noqa: E731
        return Step(i32(cu), i32(lens), i32([r + [0] * (width - len(r)) for r in rows]).view(len(rows), width), i32(who),
                    i32(pos), torch.tensor(slots, dtype=torch.int64).to(self.device),
                    max([n for _, n in requests] + [0]), max(lens + [0]), cu[-1])


@dataclass
class Adapters:
    """Every adapter's low-rank pair beside one projection: a [adapters, rank, K], b [adapters, N, rank]."""

    a: torch.Tensor
    b: torch.Tensor
    scale: torch.Tensor                    # fp32 [adapters]
    ranks: Optional[torch.Tensor] = None   # int32 [adapters]


@dataclass
class BatchedBlock:
    """A transformer block (src/nn.c:579-700) on packed weights for ragged batches.  Weights are ``QWeight`` [N, K]:
    wq, wk, wv, wo, and SwiGLU's gate w1, down w2 and up w3; norm weights fp32.  ``residual_scale`` multiplies both
    branches before they join the residual stream (1 in the reference).  ``adapters`` maps any of wq, wk, wv, wo and w2
    to its ``Adapters``; the gated pair w1, w3 runs fused and takes none."""

    wq: QWeight
    wk: QWeight
    wv: QWeight
    wo: QWeight
    w1: QWeight
    w2: QWeight
    w3: QWeight
    norm_attn: torch.Tensor
    norm_ffn: torch.Tensor
    heads: int
    kv_heads: int
    eps: float = 1e-5
    residual_scale: float = 1.0
    causal: bool = True
    adapters: Optional[Dict[str, Adapters]] = None

    def __post_init__(self):
        bad = set(self.adapters or ()) - {"wq", "wk", "wv", "wo", "w2"}
        if bad:
            raise ValueError(f"no adapters beside {sorted(bad)}")

    def _project(self, name: str, x, step: Step):
        y = matmul_nt_q(x, getattr(self, name))
        ad = (self.adapters or {}).get(name)
        return y if ad is None else lora(x, ad.a, ad.b, step.cu, step.adapter, ad.scale, base=y, out=y, ranks=ad.ranks)

    def __call__(self, h, n, step: Step, cache: PagedCache, layer: int, freqs=None, next_norm=None):
        """h [tokens, D] fp32, the residual stream; n = RMSNorm(h) * norm_attn.  Returns the block's output and, with
        next_norm, its norm (else None)."""
        hd = self.wq.N // self.heads
        q = self._project("wq", n, step).view(-1, self.heads, hd)
        k = self._project("wk", n, step).view(-1, self.kv_heads, hd)
        v = self._project("wv", n, step).view(-1, self.kv_heads, hd)
        ck, cv = cache.k[layer], cache.v[layer]
        q = rope_append(q, k, v, freqs, step.positions, step.slots, ck, cv)
        a = paged_attention(q, ck, cv, step.table, step.cu, step.kv_len, step.max_q, step.max_kv, causal=self.causal,
                            out_dtype=torch.float32)
        o = self._project("wo", a.view(-1, self.heads * hd), step)
        h, n = norm_residual(o, h, self.norm_ffn, alpha=self.residual_scale, eps=self.eps)
        g = matmul_nt_q(n, self.w1, up=self.w3)
        return norm_residual(self._project("w2", g, step), h, next_norm, alpha=self.residual_scale, eps=self.eps)


__all__ = ["Step", "PagedCache", "Adapters", "BatchedBlock"]
