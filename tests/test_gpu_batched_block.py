"""BatchedBlock: several utterances in one ragged batch, over several steps, against the float64 block of
tests/test_gpu_block.py run for each utterance alone, with and without adapters."""
from __future__ import annotations

import numpy as np
import pytest

torch = pytest.importorskip("torch")
import voxq  # noqa: E402
from test_gpu_block import block_ref, exact_weight, rmsnorm  # noqa: E402
from voxq.batched_block import Adapters, BatchedBlock, PagedCache  # noqa: E402

pytestmark = pytest.mark.gpu

# |out - ref| <= TOL (|ref| + rms(ref)): the projections' own bound (fp16 operands above 8 rows, 5e-3 per product
# relative to sum |w x| / sqrt(K), against the sum of five of them in the output) plus, for a bf16 cache, a rounding of
# 2^-9 of q, k, v and the weights
TOL = {torch.float32: 5e-3, torch.bfloat16: 2e-2}


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("with_adapters", [False, True], ids=["plain", "adapters"])
def test_batched_block_matches_each_utterance_alone(dtype, with_adapters):
    rng = np.random.default_rng(7)
    D, H, KVH, hd, F, eps = 256, 8, 2, 64, 512, 1e-6
    shapes = {"wq": (H * hd, D), "wk": (KVH * hd, D), "wv": (KVH * hd, D), "wo": (D, H * hd), "w1": (F, D), "w2": (D, F), "w3": (F, D)}
    W = {k: exact_weight(rng, *s, "q8") for k, s in shapes.items()}
    for k in ("n1", "n2"):
        W[k] = (1.0 + 0.1 * rng.standard_normal(D)).astype(np.float32)
    dev = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
    ads, delta = {}, {}
    if with_adapters:
        for k in ("wq", "wv", "wo", "w2"):
            N, K = shapes[k]
            a, b = rng.standard_normal((2, 8, K)).astype(np.float32) * K ** -0.5, rng.standard_normal((2, N, 8)).astype(np.float32) * 0.1
            ads[k] = Adapters(dev(a), dev(b), torch.tensor([1.0, 0.5], device="cuda"))
            delta[k] = [s * (b[i] @ a[i]) for i, s in enumerate((1.0, 0.5))]
    block = BatchedBlock(**{k: voxq.QWeight.from_float(dev(W[k]), voxq.Q8) for k in shapes}, norm_attn=dev(W["n1"]),
                         norm_ffn=dev(W["n2"]), heads=H, kv_heads=KVH, eps=eps, adapters=ads)
    freqs = voxq.rope_freqs(600, hd)
    fr = freqs.cpu().numpy().astype(np.float64)
    cache = PagedCache(1, 60, 16, KVH, hd, dtype=dtype)
    voice = {"a": 0, "c": 1}
    ref = {}
    for s in "abc":
        w = dict(W)
        for k in delta:
            if s in voice:
                w[k] = W[k] + delta[k][voice[s]]
        ref[s] = (w, np.zeros((1, KVH, 600, hd)), np.zeros((1, KVH, 600, hd)))
    pos = {s: 0 for s in "abc"}
    for ask in ([("a", 37), ("b", 5)], [("b", 1), ("c", 130), ("a", 1)], [("a", 1), ("b", 1), ("c", 1)], [("c", 20), ("b", 0), ("a", 2)]):
        step = cache.step(ask, voice)
        x = rng.standard_normal((step.tokens, D)).astype(np.float32)
        h0 = dev(x)
        n0 = voxq.norm_residual(h0, h0, block.norm_attn, alpha=0.0, eps=eps)[1]
        h, n = block(h0, n0, step, cache, 0, freqs, next_norm=block.norm_attn)
        at = 0
        for s, k in ask:
            if k == 0:
                continue
            w, ck, cv = ref[s]
            i = np.arange(k)[:, None] + pos[s]
            mask = np.where(np.arange(pos[s] + k)[None] <= i, 0.0, -np.inf)
            y = block_ref(x[None, at:at + k], w, ck, cv, mask, fr, pos[s], H, KVH, hd, eps)[0]
            for got, want in ((h, y), (n, rmsnorm(y, W["n1"], eps))):
                g = got[at:at + k].cpu().numpy().astype(np.float64)
                err = np.abs(g - want) / (np.abs(want) + np.sqrt((want ** 2).mean()))
                assert np.isfinite(g).all() and err.max() <= TOL[dtype], f"{ask} {s}: {err.max():.2e}"
            pos[s] += k
            at += k
    assert int(voxq.lib().voxq_device_error(1)) == 0
