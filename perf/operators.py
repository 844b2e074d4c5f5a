"""The operators of a batched decoder step, as cases to time: rotary positions written into a paged KV cache,
attention of each sequence's new tokens over that cache, low-rank adapters of many requests beside a shared
projection, and the norms around a block fused with its gate and residual scale.

`run` makes the library's calls where `own` is true and otherwise computes the same in elementary torch
operations in fp32, rounded once at the end.  Lengths are part of the case (drawn from its "mix"), values come
from the seed."""
import itertools
import math
import os
import random
import sys

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}


def _voxq():
    root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "voxcpm2-c_b200")
    if root not in sys.path:
        sys.path.insert(0, root)
    import voxq
    return voxq


# ---------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------

def listed():
    return [
        # one utterance's next token on a short context (16 query / 2 kv heads x 64): latency alone
        {"name": "attn_step_one", "op": "attn", "b": 1, "q_lo": 1, "q_hi": 1, "past_lo": 516, "past_hi": 516,
         "heads": 16, "kv_heads": 2, "dim": 64, "page": 16, "dtype": "bf16", "causal": True, "empty": False, "mix": 1},
        # the next token of 64 utterances at once, each with its own context length
        {"name": "attn_step_batch", "op": "attn", "b": 64, "q_lo": 1, "q_hi": 1, "past_lo": 600, "past_hi": 4095,
         "heads": 16, "kv_heads": 2, "dim": 128, "page": 16, "dtype": "bf16", "causal": True, "empty": False, "mix": 2},
        # few utterances with very long contexts: too few rows for the GPU unless the keys are split
        {"name": "attn_step_long", "op": "attn", "b": 3, "q_lo": 1, "q_hi": 1, "past_lo": 14000, "past_hi": 32767,
         "heads": 16, "kv_heads": 2, "dim": 128, "page": 64, "dtype": "f16", "causal": True, "empty": False, "mix": 3},
        # the residual model's continuation late in an utterance: some 60 rows over about 12 800 cached keys
        {"name": "attn_chunk", "op": "attn", "b": 3, "q_lo": 40, "q_hi": 64, "past_lo": 11000, "past_hi": 12800,
         "heads": 16, "kv_heads": 2, "dim": 128, "page": 32, "dtype": "bf16", "causal": True, "empty": False, "mix": 4},
        # prompts of a batch, each written whole
        {"name": "attn_prefill", "op": "attn", "b": 6, "q_lo": 1500, "q_hi": 4096, "past_lo": 0, "past_hi": 0,
         "heads": 16, "kv_heads": 2, "dim": 128, "page": 64, "dtype": "bf16", "causal": True, "empty": False, "mix": 5},
        # fp32 rows that see all of their own sequence, odd lengths and pages, one sequence without rows
        {"name": "attn_f32_odd", "op": "attn", "b": 5, "q_lo": 21, "q_hi": 133, "past_lo": 300, "past_hi": 1500,
         "heads": 16, "kv_heads": 2, "dim": 64, "page": 24, "dtype": "f32", "causal": False, "empty": True, "mix": 6},
        # one token of each of 48 utterances: fp32 projections rotated and stored as bf16
        {"name": "rope_step", "op": "rope", "b": 48, "q_lo": 1, "q_hi": 1, "past_lo": 60, "past_hi": 2000, "heads": 16,
         "kv_heads": 2, "dim": 128, "rot": 128, "page": 16, "dtype": "f32", "cache": "bf16", "interleaved": False,
         "pad": 0, "mix": 7},
        # prompts: interleaved pairs over half of each head, some padding rows
        {"name": "rope_prefill", "op": "rope", "b": 7, "q_lo": 700, "q_hi": 2500, "past_lo": 0, "past_hi": 900,
         "heads": 16, "kv_heads": 4, "dim": 128, "rot": 64, "page": 32, "dtype": "bf16", "cache": "bf16",
         "interleaved": True, "pad": 37, "mix": 8},
        # the next token of 40 requests with a voice adapter each (some without) beside a fp32 projection
        {"name": "lora_step", "op": "lora", "b": 40, "q_lo": 1, "q_hi": 1, "k": 2048, "n": 2048, "rank": 16,
         "adapters": 12, "dtype": "f32", "wdtype": "bf16", "ragged_rank": False, "mix": 9},
        # prompts of requests with adapters of different ranks
        {"name": "lora_prefill", "op": "lora", "b": 9, "q_lo": 200, "q_hi": 1700, "k": 1024, "n": 4096, "rank": 32,
         "adapters": 7, "dtype": "bf16", "wdtype": "bf16", "ragged_rank": True, "mix": 10},
        # a residual stream's two rows between two layers
        {"name": "norm_step", "op": "norm", "m": 2, "d": 2048, "dtype": "f32", "post": False, "gate": "none", "mix": 11},
        # a gated block (one gate per sequence) with norms on both sides, prompt rows
        {"name": "norm_prefill", "op": "norm", "m": 8191, "d": 1024, "dtype": "bf16", "post": True, "gate": "sequence",
         "mix": 12},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _drawn(rng):
    op = rng.choice(["attn", "attn", "attn", "rope", "lora", "lora", "norm"])
    mix = rng.randrange(1 << 30)
    if op == "attn":
        kv_heads = rng.choice([1, 2, 2, 3, 4, 8])
        q_hi = rng.choice([1, 1, _log_int(rng, 2, 100), _log_int(rng, 100, 3000)])
        past_hi = _log_int(rng, 20, 30000) if q_hi < 200 else rng.choice([0, _log_int(rng, 20, 8000)])
        return {"op": op, "b": _log_int(rng, 1, 64), "q_lo": max(1, q_hi // rng.choice([1, 2, 5])), "q_hi": q_hi,
                "past_lo": past_hi // rng.choice([1, 2, 7]), "past_hi": past_hi,
                "heads": kv_heads * rng.choice([1, 2, 4, 6, 8, 8]), "kv_heads": kv_heads,
                "dim": rng.choice([64, 128, 128, 80, 256]), "page": rng.choice([8, 16, 16, 24, 32, 64, 128]),
                "dtype": rng.choice(["f32", "f16", "bf16", "bf16"]), "causal": rng.random() < 0.7,
                "empty": rng.random() < 0.2, "mix": mix}
    if op == "rope":
        dim = rng.choice([64, 128, 128, 80, 256])
        dtype = rng.choice(["f32", "f16", "bf16"])
        q_hi = rng.choice([1, _log_int(rng, 2, 3000)])
        return {"op": op, "b": _log_int(rng, 1, 100), "q_lo": max(1, q_hi // 3), "q_hi": q_hi, "past_lo": 0,
                "past_hi": _log_int(rng, 10, 4000), "heads": rng.choice([4, 8, 14, 16, 32]),
                "kv_heads": rng.choice([1, 2, 4, 8]), "dim": dim, "rot": rng.choice([dim, dim, dim // 2]),
                "page": rng.choice([8, 16, 24, 64]), "dtype": dtype,
                "cache": rng.choice(["f32", "f16", "bf16"]) if dtype == "f32" else dtype,
                "interleaved": rng.random() < 0.4, "pad": rng.choice([0, 0, _log_int(rng, 1, 50)]), "mix": mix}
    if op == "lora":
        dtype = rng.choice(["f32", "f16", "bf16", "bf16"])
        q_hi = rng.choice([1, _log_int(rng, 2, 2000)])
        return {"op": op, "b": _log_int(rng, 1, 100), "q_lo": max(1, q_hi // 4), "q_hi": q_hi,
                "k": 8 * _log_int(rng, 32, 768), "n": 8 * _log_int(rng, 16, 768), "rank": rng.choice([8, 16, 16, 32, 64]),
                "adapters": rng.randint(1, 16), "dtype": dtype,
                "wdtype": rng.choice(["f32", "f16", "bf16"]) if dtype == "f32" else dtype,
                "ragged_rank": rng.random() < 0.5, "mix": mix}
    return {"op": op, "m": _log_int(rng, 1, 8191), "d": rng.choice([8 * _log_int(rng, 8, 512), _log_int(rng, 64, 4096)]),
            "dtype": rng.choice(["f32", "f16", "bf16"]), "post": rng.random() < 0.5,
            "gate": rng.choice(["none", "one", "sequence"]), "mix": mix}


def _cost(case):
    w = work(case)
    return w["bytes"] / 6e12 + w["flops"] / (5e13 if case.get("dtype") == "f32" else 1e15)


def _scores(case):
    n, past = _lengths(case)
    return case["b"] * case["heads"] * max(n) * max(p + q for p, q in zip(past, n))


def draw(rng):
    top = {}
    for c in listed():
        top[c["op"]] = max(top.get(c["op"], 0.0), _cost(c))
    while True:
        case = _drawn(rng)
        if _cost(case) > top[case["op"]] or case["op"] == "attn" and _scores(case) > 1.3e9:
            continue
        return case


def _lengths(case):
    """(new tokens, cached tokens before them) of every sequence: the case's own, whatever the seed."""
    rng = random.Random(case["mix"])
    n = [_log_int(rng, case["q_lo"], case["q_hi"]) for _ in range(case["b"])]
    past = [int(rng.uniform(case.get("past_lo", 0), case.get("past_hi", 0) + 0.999)) for _ in range(case["b"])]
    if case.get("empty") and case["b"] > 1:
        n[1] = 0
    return n, past


def _adapters(case):
    """Each request's adapter (-1: none) and each adapter's rank."""
    rng = random.Random(case["mix"] + 1)
    who = [rng.randint(0, case["adapters"] - 1) if rng.random() < 0.85 else -1 for _ in range(case["b"])]
    ranks = [rng.choice([case["rank"], max(1, case["rank"] // 2), max(1, case["rank"] // 3)]) if case["ragged_rank"] else case["rank"]
             for _ in range(case["adapters"])]
    return who, ranks


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------

def _ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype).to("cuda")


def _starts(n):
    return [0, *itertools.accumulate(n)]


def _table(rng, lens, page):
    """Block table rows in a random order of the pool's pages; page 0 belongs to no sequence."""
    need = [max(1, -(-x // page)) for x in lens]
    pages = list(range(1, 1 + sum(need)))
    rng.shuffle(pages)
    return [pages[at:at + c] + [0] * (max(need) - c) for at, c in zip(_starts(need), need)], 1 + sum(need)


def _freqs(n_pos, rot):
    """cos and sin of position * 10000^(-2i/rot), [n_pos, rot/2, 2]."""
    inv = 10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64, device="cuda") / rot)
    ang = torch.arange(n_pos, dtype=torch.float64, device="cuda")[:, None] * inv[None, :]
    return torch.stack([ang.cos(), ang.sin()], dim=-1).float().contiguous()


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rng = random.Random(seed)
    dt = DTYPES[case["dtype"]]

    def normal(*shape, scale=1.0, dtype=dt):
        return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)

    s = {"op": case["op"]}
    if case["op"] == "attn":
        n, past = _lengths(case)
        lens = [a + b for a, b in zip(n, past)]
        rows, pages = _table(rng, lens, case["page"])
        h, kvh, d = case["heads"], case["kv_heads"], case["dim"]
        # projections of normed rows: unit variance, keys and values with a mean per channel
        mean = torch.randn(1, 1, kvh, d, generator=g, device="cuda")
        s["k"] = (torch.randn(pages, case["page"], kvh, d, generator=g, device="cuda") + 0.5 * mean).to(dt)
        s["v"] = (torch.randn(pages, case["page"], kvh, d, generator=g, device="cuda") + 0.2 * mean).to(dt)
        s["q"] = normal(sum(n), h, d, scale=1.5)
        s["table"], s["cu"], s["kv_len"] = _ints(rows), _ints(_starts(n)), _ints(lens)
        s["max_q"], s["max_kv"], s["causal"] = max(n), max(lens), case["causal"]
    elif case["op"] == "rope":
        n, past = _lengths(case)
        rows, pages = _table(rng, [a + b for a, b in zip(n, past)], case["page"])
        h, kvh, d, page, ct = case["heads"], case["kv_heads"], case["dim"], case["page"], DTYPES[case["cache"]]
        pos = [p + i for a, p in zip(n, past) for i in range(a)]
        slot = [rows[j][(p + i) // page] * page + (p + i) % page for j, (a, p) in enumerate(zip(n, past)) for i in range(a)]
        pos, slot = pos + [0] * case["pad"], slot + [-1] * case["pad"]
        qkv = normal(len(pos), (h + 2 * kvh) * d)  # one projection's output, as a fused QKV product gives it
        s["q"] = qkv[:, :h * d].unflatten(1, (h, d))
        s["k"] = qkv[:, h * d:(h + kvh) * d].unflatten(1, (kvh, d))
        s["v"] = qkv[:, (h + kvh) * d:].unflatten(1, (kvh, d))
        s["cache_k"], s["cache_v"] = normal(pages, page, kvh, d, dtype=ct), normal(pages, page, kvh, d, dtype=ct)
        s["freqs"] = _freqs(max(pos) + 1, case["rot"])
        s["pos"], s["slot"], s["interleaved"] = _ints(pos), _ints(slot, torch.int64), case["interleaved"]
    elif case["op"] == "lora":
        n, _ = _lengths(case)
        who, ranks = _adapters(case)
        k, m, r, wt = case["k"], case["n"], case["rank"], DTYPES[case["wdtype"]]
        s["x"], s["base"] = normal(sum(n), k), normal(sum(n), m)
        s["a"] = normal(case["adapters"], r, k, scale=k ** -0.5, dtype=wt)
        s["b"] = normal(case["adapters"], m, r, scale=r ** -0.5, dtype=wt)
        s["cu"], s["who"], s["ranks"] = _ints(_starts(n)), _ints(who), _ints(ranks)
        s["scale"] = 0.25 + torch.rand(case["adapters"], generator=g, device="cuda")
    else:
        m, d = case["m"], case["d"]
        s["y"], s["x"] = normal(m, d, scale=0.7), normal(m, d, scale=1.3)
        s["w_pre"] = 1 + normal(d, scale=0.1, dtype=torch.float32)
        s["w_post"] = 1 + normal(d, scale=0.1, dtype=torch.float32) if case["post"] else None
        rows = {"none": 0, "one": 1, "sequence": max(1, m // 300)}[case["gate"]]
        s["gate"] = normal(rows, d) if rows else None
        s["gate_index"] = _ints(sorted(rng.randrange(rows) for _ in range(m))) if rows > 1 else None
        s["alpha"], s["eps"] = 1.4 / math.sqrt(24), 1e-5
    return s


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------

def run(s):
    if own:
        return _own(s)
    return {"attn": _plain_attn, "rope": _plain_rope, "lora": _plain_lora, "norm": _plain_norm}[s["op"]](s)


def _own(s):
    v = _voxq()
    if s["op"] == "attn":
        return v.paged_attention(s["q"], s["k"], s["v"], s["table"], s["cu"], s["kv_len"], s["max_q"], s["max_kv"],
                                 causal=s["causal"])
    if s["op"] == "rope":
        q = v.rope_append(s["q"], s["k"], s["v"], s["freqs"], s["pos"], s["slot"], s["cache_k"], s["cache_v"],
                          interleaved=s["interleaved"])
        return q, s["cache_k"], s["cache_v"]
    if s["op"] == "lora":
        return v.lora(s["x"], s["a"], s["b"], s["cu"], s["who"], s["scale"], base=s["base"], ranks=s["ranks"])
    return v.norm_residual(s["y"], s["x"], s["w_pre"], w_post=s["w_post"], gate=s["gate"], gate_index=s["gate_index"],
                           alpha=s["alpha"], eps=s["eps"])


def _plain_attn(s):
    q, kc, vc, cu, kv_len = s["q"].float(), s["k"], s["v"], s["cu"].long(), s["kv_len"].long()
    t, h, d = q.shape
    page, kvh = kc.shape[1], kc.shape[2]
    b, nq, nk, grp = len(kv_len), s["max_q"], s["max_kv"], h // kc.shape[2]
    n = cu[1:] - cu[:-1]
    pos, row = torch.arange(nk, device="cuda"), torch.arange(nq, device="cuda")
    slot = s["table"].long()[:, pos // page] * page + pos % page                        # [b, nk]
    k, v = kc.flatten(0, 1)[slot].float(), vc.flatten(0, 1)[slot].float()               # [b, nk, kvh, d]
    qp = q[(cu[:-1, None] + row).clamp(max=t - 1)]                                      # [b, nq, h, d]
    qp = qp.unflatten(2, (kvh, grp)).permute(0, 2, 3, 1, 4).reshape(b, kvh, grp * nq, d)
    sc = (qp @ k.permute(0, 2, 3, 1)).view(b, kvh, grp, nq, nk) * d ** -0.5
    seen = pos[None, None, :] < kv_len[:, None, None]                                   # [b, 1 or nq, nk]
    if s["causal"]:
        seen = seen & (pos[None, None, :] <= (kv_len - n)[:, None, None] + row[None, :, None])
    sc = sc.masked_fill_(~seen[:, None, None], float("-inf"))
    p = (sc - sc.amax(-1, keepdim=True).clamp(min=-3e38)).exp_()
    total = p.sum(-1, keepdim=True)
    o = (p.view(b, kvh, grp * nq, nk) @ v.permute(0, 2, 1, 3)).view(b, kvh, grp, nq, d) / total.clamp(min=1e-30)
    o = o.permute(0, 3, 1, 2, 4).reshape(b, nq, h, d)
    tok = torch.arange(t, device="cuda")
    own_seq = (tok[:, None] >= cu[None, 1:]).sum(1)
    return o[own_seq, tok - cu[own_seq]].to(s["q"].dtype)


def _plain_rotate(x, freqs, pos, interleaved):
    x, cs = x.float(), freqs[pos.long()][:, None]
    half = cs.shape[2]
    c, sn = cs[..., 0], cs[..., 1]
    if interleaved:
        a, b = x[..., 0:2 * half:2], x[..., 1:2 * half:2]
        turned = torch.stack([a * c - b * sn, a * sn + b * c], dim=-1).flatten(-2)
    else:
        a, b = x[..., :half], x[..., half:2 * half]
        turned = torch.cat([a * c - b * sn, a * sn + b * c], dim=-1)
    return torch.cat([turned, x[..., 2 * half:]], dim=-1)


def _plain_rope(s):
    ck, cv = s["cache_k"], s["cache_v"]
    fk, fv = ck.flatten(0, 1), cv.flatten(0, 1)
    live, at = (s["slot"] >= 0)[:, None, None], s["slot"].clamp(min=0)  # slot 0 is never a sequence's
    k = _plain_rotate(s["k"], s["freqs"], s["pos"], s["interleaved"]).to(ck.dtype)
    fk.index_copy_(0, at, torch.where(live, k, fk[at]))
    fv.index_copy_(0, at, torch.where(live, s["v"].to(cv.dtype), fv[at]))
    return _plain_rotate(s["q"], s["freqs"], s["pos"], s["interleaved"]).to(ck.dtype), ck, cv


def _plain_lora(s):
    a, b, cu = s["a"].float(), s["b"].float(), s["cu"].long()
    na, r, k = a.shape
    tok = torch.arange(s["x"].shape[0], device="cuda")
    who = s["who"].long()[(tok[:, None] >= cu[None, 1:]).sum(1)]                        # each row's adapter
    h = (s["x"].float() @ a.view(na * r, k).T).view(-1, na, r)
    keep = (who[:, None] == torch.arange(na, device="cuda"))[:, :, None] & \
        (torch.arange(r, device="cuda") < s["ranks"].long()[:, None])[None]
    h = torch.where(keep, h * s["scale"][None, :, None], torch.zeros((), device="cuda")).view(-1, na * r)
    return (s["base"].float() + h @ b.permute(0, 2, 1).reshape(na * r, -1)).to(s["base"].dtype)


def _plain_norm(s):
    z = s["y"].float()
    if s["w_post"] is not None:
        z = z * torch.rsqrt(z.square().mean(-1, keepdim=True) + s["eps"]) * s["w_post"]
    if s["gate"] is not None:
        g = s["gate"].float()
        z = z * (g if s["gate_index"] is None else g[s["gate_index"].long()])
    h = s["x"].float() + s["alpha"] * z
    n = h * torch.rsqrt(h.square().mean(-1, keepdim=True) + s["eps"]) * s["w_pre"]
    return h.to(s["x"].dtype), n.to(s["x"].dtype)


# ---------------------------------------------------------------------------
# What a pass cannot do without
# ---------------------------------------------------------------------------

def work(case):
    e = SIZE[case["dtype"]]
    if case["op"] == "attn":
        n, past = _lengths(case)
        h, kvh, d = case["heads"], case["kv_heads"], case["dim"]
        seen = sum(a * p + (a * (a + 1) // 2 if case["causal"] else a * a) for a, p in zip(n, past))
        keys = sum(a + p for a, p in zip(n, past) if a)
        tables = sum(-(-(a + p) // case["page"]) * 4 for a, p in zip(n, past) if a)
        return {"bytes": 2 * sum(n) * h * d * e + 2 * keys * kvh * d * e + tables + 8 * len(n), "flops": 4 * seen * h * d}
    if case["op"] == "rope":
        n, past = _lengths(case)
        h, kvh, d, ce, t = case["heads"], case["kv_heads"], case["dim"], SIZE[case["cache"]], sum(n)
        places = len({p + i for a, p in zip(n, past) for i in range(a)})
        return {"bytes": t * (h + 2 * kvh) * d * (e + ce) + case["pad"] * h * d * (e + ce) + places * case["rot"] * 4 + 12 * (t + case["pad"]),
                "flops": 3 * t * (h + kvh) * case["rot"]}
    if case["op"] == "lora":
        n, _ = _lengths(case)
        who, ranks = _adapters(case)
        k, m, we = case["k"], case["n"], SIZE[case["wdtype"]]
        rows = sum(n)
        adapted = [(a, ranks[w]) for a, w in zip(n, who) if w >= 0]
        weights = sum(ranks[w] for w in set(who) if w >= 0) * (k + m) * we
        return {"bytes": sum(a for a, _ in adapted) * k * e + 2 * rows * m * e + weights,
                "flops": sum(2 * a * r * (k + m) for a, r in adapted) + rows * m}
    m, d = case["m"], case["d"]
    rows = {"none": 0, "one": 1, "sequence": max(1, m // 300)}[case["gate"]]
    return {"bytes": 4 * m * d * e + rows * d * e + (2 if case["post"] else 1) * d * 4 + (4 * m if rows > 1 else 0),
            "flops": m * d * (10 if case["post"] else 6)}


# ---------------------------------------------------------------------------
# From the definition, in 64 bits
# ---------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    f8 = torch.float64
    if case["op"] == "attn":
        n, past = _lengths(case)
        q, kc, vc = s["q"].to(f8), s["k"], s["v"]
        out, at, grp = torch.zeros_like(q), 0, case["heads"] // case["kv_heads"]
        for j, (a, p) in enumerate(zip(n, past)):
            if a == 0:
                continue
            pages = s["table"][j, :-(-(a + p) // case["page"])].long()
            keys, vals = (c[pages].flatten(0, 1)[:a + p].to(f8) for c in (kc, vc))
            for head in range(case["heads"]):
                dots = torch.einsum("id,jd->ij", q[at:at + a, head], keys[:, head // grp]) / math.sqrt(case["dim"])
                if case["causal"]:
                    i, jj = torch.arange(a, device="cuda")[:, None], torch.arange(a + p, device="cuda")[None]
                    dots[jj > p + i] = -math.inf
                out[at:at + a, head] = torch.softmax(dots, dim=1) @ vals[:, head // grp]
            at += a
        return out
    if case["op"] == "rope":
        half = case["rot"] // 2

        def turn(x):
            y = x.to(f8).clone()
            cs = s["freqs"].to(f8)[s["pos"].long()]
            z = torch.complex(cs[..., 0], cs[..., 1])[:, None]
            at = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if case["interleaved"] else (slice(0, half), slice(half, 2 * half))
            z = z * torch.complex(y[..., at[0]].contiguous(), y[..., at[1]].contiguous())
            y[..., at[0]], y[..., at[1]] = z.real, z.imag
            return y

        ck, cv = s["cache_k"].to(f8), s["cache_v"].to(f8)
        live = (s["slot"] >= 0).nonzero()[:, 0]
        ck.view(-1, *ck.shape[2:])[s["slot"][live]] = turn(s["k"])[live]
        cv.view(-1, *cv.shape[2:])[s["slot"][live]] = s["v"].to(f8)[live]
        return turn(s["q"]), ck, cv
    if case["op"] == "lora":
        n, _ = _lengths(case)
        who, ranks = _adapters(case)
        out, at = s["base"].to(f8), 0
        for a, w in zip(n, who):
            if w >= 0:
                low = s["x"][at:at + a].to(f8) @ s["a"][w, :ranks[w]].to(f8).T
                out[at:at + a] += s["scale"][w].to(f8) * (low @ s["b"][w, :, :ranks[w]].to(f8).T)
            at += a
        return out

    def normed(v, w):
        return v / torch.sqrt((v * v).sum(1, keepdim=True) / v.shape[1] + s["eps"]) * w.to(f8)

    z = s["y"].to(f8)
    if s["w_post"] is not None:
        z = normed(z, s["w_post"])
    if s["gate"] is not None:
        z = z * s["gate"].to(f8)[s["gate_index"].long() if s["gate_index"] is not None else torch.zeros(len(z), dtype=torch.long, device="cuda")]
    h = s["x"].to(f8) + s["alpha"] * z
    return h, normed(h, s["w_pre"])
