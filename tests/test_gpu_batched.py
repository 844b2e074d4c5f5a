"""The operators of a batched decoder step on the GPU against plain 64-bit forms (tests/batched_ref.py, which
derives the bounds)."""
from __future__ import annotations

import math
import random

import pytest

torch = pytest.importorskip("torch")
import batched_ref as R  # noqa: E402
import voxq  # noqa: E402

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
TYPES = [F32, F16, BF16]
ids = lambda t: str(t).replace("torch.", "") if isinstance(t, torch.dtype) else None  # noqa: E731


def ints(v, dtype=torch.int32):
    return torch.tensor(list(v), dtype=dtype, device="cuda")


def starts(n):
    cu = [0]
    for a in n:
        cu.append(cu[-1] + a)
    return cu


class Pool:
    """A paged cache with random pages per sequence; every row that no sequence owns is NaN."""

    def __init__(self, lens, page, kv_heads, dim, dtype, seed=0, spare=1, layout="pshd"):
        rng = random.Random(seed)
        g = torch.Generator(device="cuda").manual_seed(seed)
        need = [-(-x // page) for x in lens]
        order = list(range(spare, spare + sum(need)))
        rng.shuffle(order)
        pages = spare + sum(need) + 1
        width = max(need + [1])
        rows = [[order.pop() for _ in range(c)] + [0] * (width - c) for c in need]
        self.table = torch.tensor(rows, dtype=torch.int32, device="cuda").view(len(lens), width)
        shape = (pages, page, kv_heads, dim)
        if layout == "phsd":  # kv heads outside the page's rows
            make = lambda: torch.full((pages, kv_heads, page, dim), math.nan, dtype=dtype, device="cuda").transpose(1, 2)  # noqa: E731
        elif layout == "wide":  # a larger row than the heads need, as in a joint K/V pool
            make = lambda: torch.full((pages, page, kv_heads + 1, dim + 16), math.nan, dtype=dtype, device="cuda")[:, :, 1:, :dim]  # noqa: E731
        else:
            make = lambda: torch.full(shape, math.nan, dtype=dtype, device="cuda")  # noqa: E731
        self.k, self.v = make(), make()
        for s, L in enumerate(lens):
            for j0 in range(0, L, page):
                c = min(page, L - j0)
                self.k[rows[s][j0 // page], :c] = torch.randn(c, kv_heads, dim, generator=g, device="cuda").to(dtype)
                self.v[rows[s][j0 // page], :c] = torch.randn(c, kv_heads, dim, generator=g, device="cuda").to(dtype)


def attend(n, lens, heads, kv_heads, dim, page, dtype, causal=True, seed=0, out_dtype=None, layout="pshd", scale=0.0,
           max_q=None, max_kv=None, q=None, **kw):
    pool = Pool(lens, page, kv_heads, dim, dtype, seed, layout=layout)
    g = torch.Generator(device="cuda").manual_seed(seed + 1)
    if q is None:
        q = torch.randn(sum(n), heads, dim, generator=g, device="cuda").to(dtype)
    cu, kv = ints(starts(n)), ints(lens)
    o = voxq.paged_attention(q, pool.k, pool.v, pool.table, cu, kv, max(n) if max_q is None else max_q,
                             max(lens) if max_kv is None else max_kv, causal=causal, scale=scale, out_dtype=out_dtype, **kw)
    ref, bound = R.attention(q, torch.nan_to_num(pool.k), torch.nan_to_num(pool.v), pool.table, cu, kv, causal,
                             scale or dim ** -0.5, out_dtype)
    R.assert_within(o, ref, bound, f"n {n} lens {lens}")
    return o


ATTN = [
    # new tokens, lengths, heads, kv heads, head dim, page
    ([1], [1], 16, 2, 64, 16),
    ([1], [517], 16, 2, 64, 16),
    ([1, 1, 1, 1], [1, 15, 16, 17], 16, 2, 128, 16),
    ([1] * 9, [3, 700, 64, 65, 1300, 127, 128, 129, 1], 16, 2, 128, 16),
    ([1, 1], [5000, 4097], 8, 1, 128, 64),
    ([1, 1], [3000, 77], 5, 5, 128, 24),
    ([3, 1, 2], [130, 64, 2], 6, 3, 80, 24),
    ([17, 0, 5], [17, 40, 300], 16, 2, 64, 7),
    ([64, 37], [1500, 900], 16, 2, 128, 32),
    ([130, 1, 257], [130, 600, 300], 8, 1, 128, 8),
    ([33, 65], [33, 65], 2, 2, 256, 128),
    ([19], [400], 12, 1, 96, 1),
    ([200, 300], [200, 811], 16, 2, 128, 64),
    ([300], [300], 32, 1, 64, 16),
]


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("causal", [True, False], ids=["causal", "full"])
@pytest.mark.parametrize("n,lens,heads,kv_heads,dim,page", ATTN)
def test_paged_attention(n, lens, heads, kv_heads, dim, page, causal, dtype):
    attend(n, lens, heads, kv_heads, dim, page, dtype, causal, seed=sum(lens) + dim)


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("dim", [8, 24, 40, 72, 120, 200, 248])
def test_paged_attention_head_dims(dim, dtype):
    attend([5, 40], [77, 140], 4, 2, dim, 16, dtype, seed=dim)


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
def test_paged_attention_rows_without_keys(dtype):
    """A sequence of length 0, one whose first rows precede its first key, and a batch of nothing but such rows."""
    o = attend([2, 5, 1], [0, 3, 0], 16, 2, 128, 16, dtype)
    assert (o[:2] == 0).all() and (o[2:4] == 0).all() and (o[4:7] != 0).any() and (o[7] == 0).all()
    pool = Pool([16], 16, 2, 64, dtype)
    q = torch.randn(300, 8, 64, device="cuda").to(dtype)
    o = voxq.paged_attention(q, pool.k, pool.v, pool.table, ints([0, 300]), ints([0]), 300, 0)
    assert (o == 0).all()


@pytest.mark.parametrize("dtype", [F16, BF16], ids=ids)
@pytest.mark.parametrize("n,lens", [([1, 1], [900, 40]), ([150, 200], [150, 333])])
def test_paged_attention_fp32_output(n, lens, dtype):
    o = attend(n, lens, 16, 2, 128, 16, dtype, out_dtype=F32)
    assert o.dtype is F32


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("layout", ["phsd", "wide"])
@pytest.mark.parametrize("n,lens", [([1, 1], [300, 41]), ([150, 200], [150, 333])])
def test_paged_attention_cache_layouts(n, lens, layout, dtype):
    attend(n, lens, 16, 2, 128, 16, dtype, layout=layout)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=ids)
@pytest.mark.parametrize("n,lens", [([1, 1], [300, 41]), ([150, 200], [150, 333])])
def test_paged_attention_strided_queries_and_loose_bounds(n, lens, dtype):
    """Queries inside a fused QKV row; max_q and max_kv above the true ones."""
    qkv = torch.randn(sum(n), 20 * 64, device="cuda").to(dtype)
    attend(n, lens, 16, 2, 64, 16, dtype, q=qkv[:, :16 * 64].unflatten(1, (16, 64)), max_q=max(n) + 70,
           max_kv=-(-max(lens) // 16) * 16)


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("n,lens", [([1, 1], [2000, 400]), ([129, 64], [129, 700])])
def test_paged_attention_large_scores(n, lens, dtype):
    """Scores of several hundred: the running maximum must carry the softmax, which becomes nearly one-hot."""
    g = torch.Generator(device="cuda").manual_seed(5)
    q = (torch.randn(sum(n), 16, 64, generator=g, device="cuda") * 64).to(dtype)
    attend(n, lens, 16, 2, 64, 16, dtype, q=q, scale=0.25)


def test_paged_attention_offsets_past_32_bits():
    """A pool of more than 2^32 bytes (and 2^31 elements): the last pages' rows are read, not wrapped ones."""
    page, kvh, dim = 64, 2, 128
    pages = (1 << 31) // (page * kvh * dim) + 40
    for dtype, n in ((BF16, [1]), (BF16, [160])):
        k = torch.zeros(pages, page, kvh, dim, dtype=dtype, device="cuda")
        v = torch.zeros_like(k)
        use = [pages - 1, 0, pages - 7]
        g = torch.Generator(device="cuda").manual_seed(3)
        for p in use:
            k[p] = torch.randn(page, kvh, dim, generator=g, device="cuda").to(dtype)
            v[p] = torch.randn(page, kvh, dim, generator=g, device="cuda").to(dtype)
        q = torch.randn(sum(n), 16, dim, generator=g, device="cuda").to(dtype)
        table, cu, kv = ints(use).view(1, 3), ints(starts(n)), ints([181])
        o = voxq.paged_attention(q, k, v, table, cu, kv, max(n), 181)
        sub = torch.tensor(use, device="cuda")
        ref, bound = R.attention(q, k[sub], v[sub], ints([0, 1, 2]).view(1, 3), cu, kv, True, dim ** -0.5)
        R.assert_within(o, ref, bound)
        del k, v


@pytest.mark.parametrize("dtype", [F16, BF16], ids=ids)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("causal", [True, False], ids=["causal", "full"])
def test_paged_attention_many_units(causal, dim, dtype):
    """More row tiles than the GPU has SMs, of very different lengths, and more sequences than one search pass takes:
    every block goes through several units."""
    rng = random.Random(dim)
    n = [700, 0, 1, 1100] + [rng.randint(1, 90) for _ in range(30)]
    attend(n, [a + rng.randint(0, 200) for a in n], 48, 3, dim, 16, dtype, causal, seed=dim)
    n = [rng.randint(9, 30) for _ in range(150)]
    attend(n, [a + rng.randint(0, 300) for a in n], 16, 2, dim, 16, dtype, causal, seed=dim)


@pytest.mark.parametrize("dtype", [F16, BF16], ids=ids)
@pytest.mark.parametrize("dim", [8, 40, 80, 120, 136, 200, 256])
@pytest.mark.parametrize("n,lens", [([700, 90, 0, 33], [1500, 90, 7, 900]), ([5] * 70, [800 + 3 * i for i in range(70)])])
def test_paged_attention_head_dims_on_many_rows(n, lens, dim, dtype):
    """Head dims below the kernels' own, in calls with enough to do for the tensor-memory kernel."""
    attend(n, lens, 18, 3, dim, 16, dtype, seed=dim)
    attend(n, lens, 18, 3, dim, 16, dtype, False, seed=dim, out_dtype=F32)


@pytest.mark.parametrize("n,lens", [([1] * 5, [3000, 20, 400, 1, 800]), ([190, 40], [300, 2500])])
def test_paged_attention_same_bits_and_other_streams(n, lens):
    """The same bits on every run, on a side stream and inside a CUDA graph."""
    pool = Pool(lens, 16, 2, 128, BF16)
    q = torch.randn(sum(n), 16, 128, device="cuda").to(BF16)
    cu, kv = ints(starts(n)), ints(lens)
    call = lambda **kw: voxq.paged_attention(q, pool.k, pool.v, pool.table, cu, kv, max(n), max(lens), **kw)  # noqa: E731
    first = call()
    assert torch.equal(first, call())
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    other = call(stream=side)
    raw = call(stream=side.cuda_stream)
    side.synchronize()
    assert torch.equal(first, other) and torch.equal(first, raw)
    graph, out = torch.cuda.CUDAGraph(), torch.empty_like(first)
    with torch.cuda.graph(graph):
        call(out=out)
    out.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(first, out)


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("batch,top", [(64, 1500), (3, 20000)])
def test_paged_attention_long_steps(batch, top, dim, dtype):
    """Next-token steps whose splits hold many more tiles than a block has stages, several times over."""
    rng = random.Random(batch)
    lens = [rng.randint(top // 3, top) for _ in range(batch)]
    pool = Pool(lens, 16, 2, dim, dtype)
    q = torch.randn(batch, 16, dim, device="cuda").to(dtype)
    cu, kv = ints(range(batch + 1)), ints(lens)
    first = None
    for _ in range(5):
        o = voxq.paged_attention(q, pool.k, pool.v, pool.table, cu, kv, 1, max(lens))
        first = o if first is None else first
        assert torch.equal(first, o)
    some = sorted(rng.sample(range(batch), min(batch, 5)))
    at = torch.tensor(some, device="cuda")
    ref, bound = R.attention(q[at], torch.nan_to_num(pool.k), torch.nan_to_num(pool.v), pool.table[at], ints(range(len(some) + 1)),
                             kv[at], True, dim ** -0.5)
    R.assert_within(first[at], ref, bound)
    assert int(voxq.lib().voxq_device_error(1)) == 0


def test_paged_attention_batch_equals_alone():
    """A sequence's step does not depend on who shares the batch, up to the split of its keys over CTAs."""
    lens = [900, 33, 2100]
    pool = Pool(lens, 16, 2, 128, F32)
    q = torch.randn(3, 16, 128, device="cuda")
    o = voxq.paged_attention(q, pool.k, pool.v, pool.table, ints([0, 1, 2, 3]), ints(lens), 1, 2100)
    for s in range(3):
        a = voxq.paged_attention(q[s:s + 1], pool.k, pool.v, pool.table[s:s + 1], ints([0, 1]), ints(lens[s:s + 1]), 1, lens[s])
        assert (a - o[s:s + 1]).abs().max() < 1e-5


# ---------------------------------------------------------------------------

ROPE_TYPES = [(F32, F32), (F32, F16), (F32, BF16), (F16, F16), (BF16, BF16)]


@pytest.mark.parametrize("dt,ct", ROPE_TYPES, ids=ids)
@pytest.mark.parametrize("inter", [False, True], ids=["half", "interleaved"])
@pytest.mark.parametrize("T,H,KVH,D,rot,page,pad", [
    (1, 16, 2, 128, 128, 16, 0), (3, 16, 2, 64, 64, 16, 0), (50, 14, 2, 64, 32, 24, 5), (37, 4, 4, 80, 40, 8, 1),
    (9, 3, 1, 256, 256, 7, 2), (5, 8, 8, 8, 8, 1, 0), (700, 16, 4, 128, 64, 32, 9), (11, 2, 2, 24, 2, 16, 0), (6, 2, 1, 72, 36, 16, 0),
    (4, 2, 1, 64, 0, 16, 0)])
def test_rope_append(T, H, KVH, D, rot, page, pad, inter, dt, ct):
    g = torch.Generator(device="cuda").manual_seed(T + D)
    pages = -(-T // page) + 3
    qkv = torch.randn(T + pad, (H + 2 * KVH) * D, generator=g, device="cuda").to(dt)
    q = qkv[:, :H * D].unflatten(1, (H, D))
    k = qkv[:, H * D:(H + KVH) * D].unflatten(1, (KVH, D))
    v = qkv[:, (H + KVH) * D:].unflatten(1, (KVH, D))
    ck = torch.randn(pages, page, KVH, D, generator=g, device="cuda").to(ct)
    cv = torch.randn(pages, page, KVH, D, generator=g, device="cuda").to(ct)
    ck0, cv0 = ck.clone(), cv.clone()
    pos = torch.randint(0, 5000, (T + pad,), generator=g, device="cuda", dtype=torch.int32)
    slot = torch.randperm(pages * page, generator=g, device="cuda")[:T + pad] if pages * page >= T + pad else None
    slot = torch.cat([torch.randperm(pages * page, generator=g, device="cuda")[:T], torch.full((pad,), -1, device="cuda")])
    freqs = voxq.rope_freqs(5000, rot) if rot else None
    qo = voxq.rope_append(q, k, v, freqs, pos, slot, ck, cv, interleaved=inter)
    fr = freqs if rot else torch.zeros(5000, 0, 2, device="cuda")
    ref, b = R.rotate(q, fr, pos, inter, ct) if rot else (R.f8(q), R.U[ct] * R.f8(q).abs() + R.TINY[ct])
    R.assert_within(qo, ref, b, "q")
    kr, kb = R.rotate(k, fr, pos, inter, ct) if rot else (R.f8(k), R.U[ct] * R.f8(k).abs() + R.TINY[ct])
    live = slot[:T].cpu()
    R.assert_within(ck.flatten(0, 1)[slot[:T]], kr[:T], kb[:T], "k")
    assert torch.equal(cv.flatten(0, 1)[slot[:T]], v[:T].to(ct))
    rest = torch.ones(pages * page, dtype=torch.bool)
    rest[live] = False
    assert torch.equal(ck.flatten(0, 1)[rest], ck0.flatten(0, 1)[rest]) and torch.equal(cv.flatten(0, 1)[rest], cv0.flatten(0, 1)[rest])


def test_rope_append_in_place_and_slots_outside():
    q, k, v = (torch.randn(4, h, 64, device="cuda") for h in (4, 2, 2))
    ck, cv = torch.zeros(2, 8, 2, 64, device="cuda"), torch.zeros(2, 8, 2, 64, device="cuda")
    freqs = voxq.rope_freqs(100, 64)
    pos, slot = ints([0, 1, 99, 7]), ints([0, 16, -5, 1 << 40], torch.int64)
    ref, b = R.rotate(q, freqs, pos, False, F32)
    out = voxq.rope_append(q, k, v, freqs, pos, slot, ck, cv, q_out=q)
    assert out is q
    R.assert_within(q, ref, b)
    assert torch.equal(cv[0, 0], v[0]) and int((cv != 0).sum()) == int((v[0] != 0).sum())
    # positions outside the table take its ends
    a = voxq.rope_append(k, k, v, freqs, ints([-3, 1000, 0, 99]), slot, ck, cv)
    c = voxq.rope_append(k, k, v, freqs, ints([0, 99, 0, 99]), slot, ck, cv)
    assert torch.equal(a, c)
    assert voxq.rope_append(q[:0], k[:0], v[:0], freqs, pos[:0], slot[:0], ck, cv).shape == (0, 4, 64)


@pytest.mark.parametrize("kw", [{}, {"scaling": "linear", "factor": 4.0}, {"scaling": "ntk", "factor": 8.0},
                                {"scaling": "yarn", "factor": 4.0, "original_len": 4096, "attn_factor": 0.1 * math.log(4.0) + 1.0},
                                {"scaling": "yarn", "factor": 16.0, "original_len": 64, "beta_fast": 8.0, "beta_slow": 2.0},
                                {"scaling": "long"}], ids=lambda k: str(k.get("scaling")) if isinstance(k, dict) else None)
@pytest.mark.parametrize("rot,theta", [(64, 10000.0), (128, 500000.0), (20, 10000.0)])
def test_rope_freqs(rot, theta, kw):
    n = 3001
    kw = dict(kw)
    i = torch.arange(rot // 2, dtype=torch.float64)
    f = theta ** (-2 * i / rot)
    if kw.get("scaling") == "linear":
        f = f / kw["factor"]
    elif kw.get("scaling") == "ntk":
        f = (theta * kw["factor"] ** (rot / (rot - 2))) ** (-2 * i / rot)
    elif kw.get("scaling") == "yarn":
        at = lambda turns: rot * math.log(kw["original_len"] / (turns * 2 * math.pi)) / (2 * math.log(theta))  # noqa: E731
        lo = min(max(math.floor(at(kw.get("beta_fast", 32.0))), 0), rot - 1)
        hi = min(max(math.ceil(at(kw.get("beta_slow", 1.0))), 0), rot - 1)
        keep = 1 - ((i - lo) / max(hi - lo, 1e-3)).clamp(0, 1)
        f = f * (1 - keep) / kw["factor"] + f * keep
    elif kw.get("scaling") == "long":
        kw["long_factors"] = [1.0 + 0.37 * j for j in range(rot // 2)]
        f = f / torch.tensor(kw["long_factors"], dtype=torch.float64)
    t = voxq.rope_freqs(n, rot, theta, **kw)
    ang = torch.arange(n, dtype=torch.float64)[:, None] * f
    ref = torch.stack([ang.cos(), ang.sin()], -1) * kw.get("attn_factor", 1.0)
    # fp32 rounding of the result; fp64 angles up to 3000 radians (a few ulps of 2^-52 each)
    R.assert_within(t, ref, 2.0 ** -24 * ref.abs() + 3001 * 2.0 ** -50)


# ---------------------------------------------------------------------------

LORA = [
    # rows per request, adapters, K, N, rank
    ([1], 1, 64, 64, 8), ([1] * 40, 12, 2048, 2048, 16), ([1, 3, 0, 2], 3, 1000, 328, 16), ([200, 17, 64, 65], 4, 1024, 512, 32),
    ([5, 70], 2, 8, 8, 64), ([33], 1, 520, 4096, 128), ([16, 15, 300], 3, 1536, 264, 24), ([0, 0, 9], 2, 256, 72, 8),
]
LORA_TYPES = [(F32, F32), (F32, F16), (F32, BF16), (F16, F16), (BF16, BF16)]


def lora_inputs(rows, nA, K, N, r, dt, wt, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed + K + N)
    x = torch.randn(sum(rows), K, generator=g, device="cuda").to(dt)
    base = torch.randn(sum(rows), N, generator=g, device="cuda").to(dt)
    a = (torch.randn(nA, r, K, generator=g, device="cuda") * K ** -0.5).to(wt)
    b = (torch.randn(nA, N, r, generator=g, device="cuda") * r ** -0.5).to(wt)
    scale = torch.rand(nA, generator=g, device="cuda") + 0.5
    rng = random.Random(seed)
    who = [rng.choice([-1] + 3 * list(range(nA))) for _ in rows]
    who[0] = 0
    return x, a, b, ints(starts(rows)), ints(who), scale, base


@pytest.mark.parametrize("dt,wt", LORA_TYPES, ids=ids)
@pytest.mark.parametrize("rows,nA,K,N,r", LORA)
def test_lora(rows, nA, K, N, r, dt, wt):
    x, a, b, cu, who, scale, base = lora_inputs(rows, nA, K, N, r, dt, wt)
    ranks = ints([max(1, r - 3 * (j % 3)) for j in range(nA)])
    for rk, bs in ((None, base), (ranks, base), (ranks, None)):
        ref, bound = R.adapters(x, a, b, cu, who, scale, bs, rk)
        R.assert_within(voxq.lora(x, a, b, cu, who, scale, base=bs, ranks=rk), ref, bound, f"ranks {rk is not None}")


@pytest.mark.parametrize("dt,wt", [(F32, F32), (F16, F16)], ids=ids)
@pytest.mark.parametrize("r", [24, 40, 64, 72])
@pytest.mark.parametrize("rows", [[1] * 50, [900, 0, 2100, 37, 1900]])
def test_lora_ranks_and_row_counts(rows, r, dt, wt):
    """Every rank class with tiles of 16 and of 64 rows."""
    test_lora(rows, 5, 328, 2184, r, dt, wt)


@pytest.mark.parametrize("dt,wt", [(F32, BF16), (BF16, BF16)], ids=ids)
@pytest.mark.parametrize("rows", [[1, 1, 1], [100, 3, 40]])
def test_lora_in_place_strided_and_unused(rows, dt, wt):
    """In place over the base, rows inside wider buffers; ranks of 0, scale 0 and adapters outside the range leave the
    base as it is; NaN in the columns past an adapter's rank are not read into the result."""
    x, a, b, cu, who, scale, base = lora_inputs(rows, 3, 256, 320, 16, dt, wt, seed=4)
    big_x = torch.zeros(sum(rows), 256 + 64, device="cuda").to(dt)
    big_x[:, 32:288] = x
    big_o = torch.full((sum(rows), 320 + 16), 7.0, device="cuda").to(dt)
    big_o[:, :320] = base
    who = ints([2, 99, 0])
    ranks = ints([0, 16, 5])
    a[2, 5:], b[2, :, 5:], a[0], b[0] = math.nan, math.nan, math.nan, math.nan
    fixed = [torch.nan_to_num(t) for t in (a, b)]
    ref, bound = R.adapters(x, *fixed, cu, who, scale, base, ranks)
    out = voxq.lora(big_x[:, 32:288], a, b, cu, who, scale, base=big_o[:, :320], out=big_o[:, :320], ranks=ranks)
    R.assert_within(out, ref, bound)
    assert torch.equal(out[rows[0]:], base[rows[0]:]) and (big_o[:, 320:] == 7).all()
    assert torch.equal(voxq.lora(x, a[:0], b[:0], cu, who, scale[:0], base=base), base)
    assert voxq.lora(x[:0], fixed[0], fixed[1], ints([0, 0]), ints([0]), scale).shape == (0, 320)


# ---------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("M,D", [(1, 1), (2, 2048), (1, 16384), (5, 1000), (3, 1001), (300, 1024), (700, 64), (4, 4100), (65, 8),
                                 (1300, 2048), (9, 16383), (2, 33), (1200, 136)])
@pytest.mark.parametrize("post,gate,pre", [(False, "none", True), (True, "index", True), (True, "one", False), (False, "rows", True)])
def test_norm_residual(M, D, post, gate, pre, dtype):
    g = torch.Generator(device="cuda").manual_seed(M + D)
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    y, x = rnd(M, D).to(dtype), (rnd(M, D) * 1.5).to(dtype)
    w_pre, w_post = 1 + 0.1 * rnd(D), 1 + 0.1 * rnd(D)
    rows = {"none": 0, "index": 4, "one": 1, "rows": M}[gate]
    gt = rnd(rows, D).to(dtype) if rows else None
    gi = torch.randint(0, 4, (M,), generator=g, device="cuda", dtype=torch.int32) if gate == "index" else None
    h, n = voxq.norm_residual(y, x, w_pre if pre else None, w_post if post else None, gt, gi, alpha=0.3, eps=1e-5)
    (hr, hb), nn = R.norm_residual(y, x, w_pre if pre else None, w_post if post else None, gt, gi, 0.3, 1e-5)
    R.assert_within(h, hr, hb, "h")
    if pre:
        R.assert_within(n, *nn, "n")
    else:
        assert n is None


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("D", [250, 258, 514, 1002, 2047, 2050, 4095, 4102, 8190, 9001])
def test_norm_residual_narrow_widths(D, dtype):
    """Widths that only two elements, or one, an access divide."""
    g = torch.Generator(device="cuda").manual_seed(D)
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    y, x, gt = rnd(37, D).to(dtype), rnd(37, D).to(dtype), rnd(1, D).to(dtype)
    w_pre, w_post = 1 + 0.1 * rnd(D), 1 + 0.1 * rnd(D)
    h, n = voxq.norm_residual(y, x, w_pre, w_post, gt, alpha=0.7, eps=1e-6)
    (hr, hb), nn = R.norm_residual(y, x, w_pre, w_post, gt, None, 0.7, 1e-6)
    R.assert_within(h, hr, hb, "h")
    R.assert_within(n, *nn, "n")


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("D,off", [(512, 0), (512, 1), (100, 3)])
def test_norm_residual_strides_and_in_place(D, off, dtype):
    """Rows of wider buffers at any alignment, in place over x and y; a gate index outside the gate takes its ends."""
    y, x = torch.randn(40, D + 8, device="cuda").to(dtype), torch.randn(40, D + 16, device="cuda").to(dtype)
    ys, xs = y[:, off:off + D], x[:, off:off + D]
    y0, x0, w = ys.clone(), xs.clone(), torch.rand(D, device="cuda") + 0.5
    gate, gi = torch.randn(3, D, device="cuda").to(dtype), ints([-2, 9] + [1] * 38)
    h, n = voxq.norm_residual(ys, xs, w, w, gate, gi, alpha=1.0, h_out=xs, n_out=ys)
    (hr, hb), nn = R.norm_residual(y0, x0, w, w, gate, gi.clamp(0, 2), 1.0, 1e-5)
    R.assert_within(xs, hr, hb, "h")
    R.assert_within(ys, *nn, "n")
    assert voxq.norm_residual(ys[:0], xs[:0], w)[1].shape == (0, D)
    z = torch.zeros(2, D, device="cuda").to(dtype)
    h, n = voxq.norm_residual(z, z, w, w)
    assert (h == 0).all() and (n == 0).all()


# ---------------------------------------------------------------------------

def test_refusals():
    pool = Pool([40], 16, 2, 64, BF16)
    q = torch.randn(1, 4, 64, device="cuda").to(BF16)
    args = (pool.table, ints([0, 1]), ints([40]), 1, 40)
    with pytest.raises(ValueError):
        voxq.paged_attention(q.float(), pool.k, pool.v, *args)
    with pytest.raises(ValueError):
        voxq.paged_attention(q, pool.k, pool.v, pool.table.long(), *args[1:])
    with pytest.raises(ValueError):
        voxq.paged_attention(q, pool.k, pool.v, *args[:-1], 49)
    with pytest.raises(voxq.VoxqError) as e:
        voxq.paged_attention(torch.zeros(1, 3, 64, device="cuda", dtype=BF16), pool.k, pool.v, *args)
    assert e.value.code == voxq.SHAPE_MISMATCH
    with pytest.raises(voxq.VoxqError) as e:
        voxq.paged_attention(torch.zeros(1, 4, 72, device="cuda", dtype=BF16)[..., 4:68], pool.k, pool.v, *args)
    assert e.value.code == voxq.UNSUPPORTED
    with pytest.raises(voxq.VoxqError) as e:
        voxq.paged_attention(q, pool.k, pool.v, *args, out=torch.empty(1, 4, 64, device="cuda", dtype=F16))
    assert e.value.code == voxq.UNSUPPORTED
    k = torch.randn(1, 2, 64, device="cuda").to(BF16)
    f = voxq.rope_freqs(50, 64)
    with pytest.raises(ValueError):
        voxq.rope_append(q, k, k, f, ints([0]), ints([0]), pool.k, pool.v)
    with pytest.raises(ValueError):
        voxq.rope_append(q, k, k.float(), f, ints([0]), ints([0], torch.int64), pool.k, pool.v)
    with pytest.raises(voxq.VoxqError) as e:
        voxq.rope_append(q, k, k, voxq.rope_freqs(50, 128), ints([0]), ints([0], torch.int64), pool.k, pool.v)
    assert e.value.code == voxq.SHAPE_MISMATCH
    x, a, b = (torch.zeros(*s, device="cuda") for s in ((2, 64), (1, 8, 64), (1, 32, 8)))
    one = torch.ones(1, device="cuda")
    with pytest.raises(ValueError):
        voxq.lora(x, a, b[:, :, :4], ints([0, 2]), ints([0]), one)
    with pytest.raises(ValueError):
        voxq.lora(x, a, b, ints([0, 2]).long(), ints([0]), one)
    with pytest.raises(voxq.VoxqError) as e:
        voxq.lora(x.to(BF16), a, b, ints([0, 2]), ints([0]), one)
    assert e.value.code == voxq.UNSUPPORTED
    with pytest.raises(voxq.VoxqError) as e:
        voxq.norm_residual(x, x, gate=torch.zeros(3, 64, device="cuda"))
    assert e.value.code == voxq.SHAPE_MISMATCH
    with pytest.raises(ValueError):
        voxq.norm_residual(x, x, one)


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("n,lens", [([1, 1], [300, 700]), ([120, 40], [300, 700])])
def test_paged_attention_fp32_is_as_close_as_fp32(n, lens, dim):
    """The error over the whole output, as a norm: 2^-20 is sixteen roundings of fp32, where single TF32 products or long
    sums inside the MMAs give more."""
    pool = Pool(lens, 16, 2, dim, F32)
    q = torch.randn(sum(n), 8, dim, device="cuda")
    cu, kv = ints(starts(n)), ints(lens)
    o = voxq.paged_attention(q, pool.k, pool.v, pool.table, cu, kv, max(n), max(lens))
    ref, _ = R.attention(q, torch.nan_to_num(pool.k), torch.nan_to_num(pool.v), pool.table, cu, kv, True, dim ** -0.5, None)
    assert float((R.f8(o) - ref).norm() / ref.norm()) < 2.0 ** -20
