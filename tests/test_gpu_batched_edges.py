"""The batched-step operators on the GPU where types, sizes and values meet their limits."""
from __future__ import annotations

import ctypes as C

import pytest

torch = pytest.importorskip("torch")
import batched_ref as R  # noqa: E402
import voxq  # noqa: E402
from test_gpu_batched import BF16, F16, F32, LORA_TYPES, Pool, ids, ints, lora_inputs, starts  # noqa: E402

pytestmark = pytest.mark.gpu

# ||out - ref|| / ||ref|| of an fp32 output over 16-bit operands.  The values have mean zero, so an error of relative size
# e in every weight gives e in this norm: weights rounded once to the operand type give their rounding's root mean square,
# 2^-8 / sqrt(12) .. 2^-7 / sqrt(12) in bf16 (over 2^-10) and 2^-13 or more in fp16; in two parts the square of that, under
# 2^-16 and 2^-22.  The bounds are 2^4 under the one and over the other for bf16, and 2^3 or more for fp16, where fp32's
# own errors (scores of 128 products: under 2^-20) are what is left.
TWO_PARTS = {BF16: 2.0 ** -13, F16: 2.0 ** -17}


@pytest.mark.parametrize("dtype", [F16, BF16], ids=ids)
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("n,lens", [([1] * 4, [64, 208, 48, 160]), ([40, 24], [64, 48]), ([48] * 70, [48, 64] * 35),
                                    ([320, 1600], [320, 1600])], ids=["step", "few", "many", "prompts"])
def test_fp32_output_keeps_the_weights_in_two_parts(n, lens, dim, dtype):
    """Whatever the size of the call, and so the kernel that runs it."""
    pool = Pool(lens, 16, 2, dim, dtype)
    q = torch.randn(sum(n), 16, dim, generator=torch.Generator(device="cuda").manual_seed(dim), device="cuda").to(dtype)
    cu, kv = ints(starts(n)), ints(lens)
    o = voxq.paged_attention(q, pool.k, pool.v, pool.table, cu, kv, max(n), max(lens), out_dtype=F32)
    ref, _ = R.attention(q, torch.nan_to_num(pool.k), torch.nan_to_num(pool.v), pool.table, cu, kv, True, dim ** -0.5, F32)
    assert float((R.f8(o) - ref).norm() / ref.norm()) < TWO_PARTS[dtype]


@pytest.mark.parametrize("dtype", [F16, BF16], ids=ids)
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_many_units_of_one_key_tile_with_odd_ends(dim, dtype):
    """Every unit of work is one tile of keys that ends inside 16 of them, so that its loader runs furthest ahead of its
    products: the same bits every time, no wait that gives up, and the right ones."""
    n = [16 + i % 3 for i in range(600)]
    lens = [a + 17 + 2 * (i % 40) for i, a in enumerate(n)]
    pool = Pool(lens, 16, 2, dim, dtype)
    q = torch.randn(sum(n), 16, dim, device="cuda").to(dtype)
    cu, kv = ints(starts(n)), ints(lens)
    outs = [voxq.paged_attention(q, pool.k, pool.v, pool.table, cu, kv, max(n), max(lens)) for _ in range(20)]
    assert all(torch.equal(outs[0], o) for o in outs) and int(voxq.lib().voxq_device_error(1)) == 0
    some = 40
    ref, bound = R.attention(q[:cu[some]], torch.nan_to_num(pool.k), torch.nan_to_num(pool.v), pool.table[:some], cu[:some + 1],
                             kv[:some], True, dim ** -0.5)
    R.assert_within(outs[0][:cu[some]], ref, bound)


@pytest.mark.parametrize("D", [8, 16, 24, 32, 48])
@pytest.mark.parametrize("H,KVH", [(1, 1), (2, 1), (1, 0), (2, 0), (0, 1)])
@pytest.mark.parametrize("rotate", [True, False], ids=["rot", "plain"])
def test_rope_append_of_few_small_heads(H, KVH, D, rotate):
    """So little a token that more tokens would fit a block than a block may have along one of its axes.  From C, where
    queries or the cache may be left out."""
    T, pages, page = 150, 21, 8
    qkv = torch.randn(T, H + 2 * KVH, D, device="cuda")
    q, k, v = qkv[:, :H], qkv[:, H:H + KVH], qkv[:, H + KVH:]
    out, ck, cv = torch.zeros(T, H, D, device="cuda"), *(torch.zeros(pages, page, KVH, D, device="cuda") for _ in range(2))
    freqs, pos = voxq.rope_freqs(200, D), ints(range(T))
    slot = torch.randperm(pages * page, device="cuda")[:T]
    row = (H + 2 * KVH) * D
    d = voxq.RopeDesc(q=q.data_ptr(), k=k.data_ptr(), v=v.data_ptr(), q_stride=row, q_head_stride=D, k_stride=row, k_head_stride=D,
                      v_stride=row, v_head_stride=D, q_out=out.data_ptr() if H else None, qo_stride=H * D, qo_head_stride=D,
                      cache_k=ck.data_ptr(), cache_v=cv.data_ptr(), page_stride=page * KVH * D, row_stride=KVH * D, head_stride=D,
                      freqs=freqs.data_ptr() if rotate else None, positions=pos.data_ptr(), slots=slot.data_ptr(), tokens=T, heads=H,
                      kv_heads=KVH, head_dim=D, rot_dim=D if rotate else 0, n_pos=200, pages=pages, page_size=page,
                      in_dtype=voxq.F32, cache_dtype=voxq.F32)
    voxq.check(voxq.lib().voxq_rope_append(C.byref(d), torch.cuda.current_stream().cuda_stream), "voxq_rope_append")
    turned = lambda x: R.rotate(x, freqs, pos, False, F32) if rotate else (R.f8(x), 0 * R.f8(x))  # noqa: E731
    if H:
        R.assert_within(out, *turned(q), "q")
    if KVH:
        R.assert_within(ck.flatten(0, 1)[slot], *turned(k), "k")
        assert torch.equal(cv.flatten(0, 1)[slot], v)


def test_flags_that_have_no_truth_value():
    """Their own error, before anything is launched."""
    class Neither:
        def __bool__(self):
            raise ArithmeticError("neither")

    pool = Pool([40], 16, 2, 64, BF16)
    q = torch.zeros(1, 4, 64, device="cuda", dtype=BF16)
    with pytest.raises(ArithmeticError):
        voxq.paged_attention(q, pool.k, pool.v, pool.table, ints([0, 1]), ints([40]), 1, 40, causal=Neither())
    with pytest.raises(ArithmeticError):
        voxq.rope_append(q, q[:, :2], q[:, :2], voxq.rope_freqs(4, 64), ints([0]), ints([0], torch.int64), pool.k, pool.v, interleaved=Neither())


def attention_by_the_formula(q, ck, cv, table, cu, kv_len, out_dtype):
    """(result, bound) in float64, causal, each row over the keys that it sees and no others, so that what is not finite
    is so by the formula."""
    u = 0.0 if q.dtype is F32 else R.U[q.dtype]
    uo = R.U[out_dtype or q.dtype]
    q, ck, cv, table = R.f8(q), R.f8(ck), R.f8(cv), table.cpu().long()
    D, page, G = q.shape[2], ck.shape[1], q.shape[1] // ck.shape[2]
    out, bound = torch.zeros_like(q), torch.zeros_like(q)
    for s, L in enumerate(kv_len.tolist()):
        lo, hi = int(cu[s]), int(cu[s + 1])
        pos = torch.arange(L)
        at = table[s, pos // page] * page + pos % page
        for i in range(hi - lo):
            see = max(min(L - (hi - lo) + i + 1, L), 0)
            if see == 0:
                continue
            for h in range(q.shape[1]):
                k, v, x = ck.flatten(0, 1)[at[:see], h // G], cv.flatten(0, 1)[at[:see], h // G], q[lo + i, h]
                sc = (k @ x) * D ** -0.5
                p = torch.softmax(sc, 0)
                fine = torch.nan_to_num(v, 0, 0, 0).abs()
                out[lo + i, h] = (p[:, None] * v).sum(0)
                delta = (torch.nan_to_num(k, 0, 0, 0).abs() @ x.abs()).amax() * D ** -0.5 * (D + 4) * R.E
                bound[lo + i, h] = uo * out[lo + i, h].abs() + (2 * u + 4 * delta + (L + 8) * R.E) * (torch.nan_to_num(p)[:, None] * fine).sum(0)
    return out, bound


@pytest.mark.parametrize("dtype,out_dtype", [(F32, None), (F16, None), (F16, F32), (BF16, None), (BF16, F32)], ids=ids)
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("rows,more", [(4, 0), (12, 0), (40, 60)], ids=["step", "few", "many"])
def test_attention_that_meets_infinities_and_nan(rows, more, dim, dtype, out_dtype):
    """Infinite and NaN keys and values, seen and not seen, give what the formula gives in every kernel: not finite where it
    is not, and unharmed elsewhere."""
    inf, nan = float("inf"), float("nan")
    # sequence: 0, 1 values, 2 keys, 3 its last token, 4 fewer keys than rows, 5 a single key, 6 on unharmed
    n = [rows] * 5 + [1] + [rows] * (1 + more)
    lens = [200, 150, 130, rows + 40, rows - 2, 1] + [rows + 24] * (1 + more)
    pool = Pool(lens, 16, 2, dim, dtype, seed=3)
    g = torch.Generator(device="cuda").manual_seed(4)
    q = torch.randn(sum(n), 8, dim, generator=g, device="cuda")
    cu = starts(n)
    q[cu[2]:cu[3], :, 5] = q[cu[2]:cu[3], :, 5].abs() + 0.1
    q[cu[2] + 1, :, 5] *= -1
    q[cu[1], 3, 7] = inf
    q[cu[5], :, 2] = 1e-37 if dtype is F32 else 0
    q = q.to(dtype)
    top = torch.finfo(dtype).max

    def put(cache, s, j, kvh, dims, value):
        cache[int(pool.table[s, j // 16]), j % 16, kvh, dims] = value
    put(pool.v, 0, 3, 0, 9, inf)
    put(pool.v, 0, 100, 0, 10, -inf)
    put(pool.v, 0, 101, 0, 11, nan)
    put(pool.v, 0, 7, 0, 12, inf)
    put(pool.v, 0, 150, 0, 12, -inf)
    put(pool.v, 1, lens[1] - 2, 1, slice(0, 40), inf)   # not seen by the first rows
    put(pool.k, 2, 20, 0, 5, -inf)                      # weight 0; a NaN for the row whose query is negative there
    put(pool.k, 2, 90, 0, 5, -inf)
    put(pool.k, 3, lens[3] - 1, 0, slice(None), nan)    # seen by the last row alone
    put(pool.v, 3, lens[3] - 1, 1, slice(None), nan)
    put(pool.v, 4, 0, 0, slice(None), nan)
    put(pool.v, 4, 1, 1, 3, -inf)
    put(pool.v, 5, 0, 0, slice(0, 8), top)
    put(pool.k, 5, 0, 1, 2, top)
    cu, kv = ints(cu), ints(lens)
    o = voxq.paged_attention(q, pool.k, pool.v, pool.table, cu, kv, max(n), max(lens), out_dtype=out_dtype)
    some = 8
    ref, bound = attention_by_the_formula(q[:int(cu[some - 1])], pool.k, pool.v, pool.table, cu[:some], kv[:some - 1], out_dtype)
    y = R.f8(o)[:ref.shape[0]]
    assert torch.equal(torch.isnan(y), torch.isnan(ref)), "NaN in other places than the formula's"
    fine = torch.isfinite(ref)
    assert torch.equal(y[~fine & ~torch.isnan(ref)], ref[~fine & ~torch.isnan(ref)]), "infinities in other places than the formula's"
    R.assert_within(torch.where(fine, y, 0.0), torch.where(fine, ref, 0.0), torch.where(fine, bound, 0.0) + R.TINY[out_dtype or dtype])
    assert torch.isfinite(o[int(cu[6]):]).all() and int(voxq.lib().voxq_device_error(1)) == 0


def test_units_of_work_that_last_long():
    """Every unit of 32 tokens ends in one with a NaN that the others do not see, so that its rows are taken again one by one:
    units of some 0.1 s, several a block, whose waits must not give up."""
    n, dim = [4100, 4096, 3000], 128
    pool = Pool(n, 16, 2, dim, BF16, seed=8)
    q = torch.randn(sum(n), 16, dim, generator=torch.Generator(device="cuda").manual_seed(8), device="cuda").to(BF16)
    args = (pool.table, ints(starts(n)), ints(n), max(n), max(n))
    clean = voxq.paged_attention(q, pool.k, pool.v, *args)
    want = torch.zeros(sum(n), dim, dtype=torch.bool)
    for s, c in enumerate(n):
        for j in range(31, c, 32):
            pool.v[int(pool.table[s, j // 16]), j % 16, :, j // 32 % dim] = float("nan")
            want[starts(n)[s] + j:starts(n)[s + 1], j // 32 % dim] = True
    o = voxq.paged_attention(q, pool.k, pool.v, *args)
    assert int(voxq.lib().voxq_device_error(1)) == 0
    assert torch.equal(torch.isnan(o).cpu(), want[:, None].expand(-1, 16, -1))
    # p rounded or not, the output rounded: 2^-8 of the value and 2^-8 of what the weights' errors move
    off = (o.float() - clean.float()).abs().cpu()[~torch.isnan(o).cpu()]
    size = clean.float().abs().cpu()[~torch.isnan(o).cpu()]
    assert (off <= 2.0 ** -7 * (size + 1.0)).all()


@pytest.mark.parametrize("dt,wt", LORA_TYPES, ids=ids)
@pytest.mark.parametrize("rows", [[5, 1], [9000, 3]], ids=["few", "many"])
def test_lora_keeps_a_nan_in_its_weights(rows, dt, wt):
    """One in A reaches every column of its request, one in B its own column; whatever its bits."""
    x, a, b, cu, _, scale, base = lora_inputs(rows, 2, 264, 520, 40, dt, wt, seed=6)
    clean = voxq.lora(x, a, b, cu, ints([0, 1]), scale, base=base)
    b[0, 300, 2] = float("nan")
    b[1].view(torch.int32 if wt is F32 else torch.int16)[7, 0] = 0x7fffffff if wt is F32 else 0x7fff
    y = voxq.lora(x, a, b, cu, ints([0, 1]), scale, base=base)
    want = torch.zeros_like(y, dtype=torch.bool)
    want[:rows[0], 300], want[rows[0]:, 7] = True, True
    assert torch.equal(torch.isnan(y), want) and torch.equal(y[~want], clean[~want])
    a[0].view(torch.int32 if wt is F32 else torch.int16)[39, 263] = 0x7fffffff if wt is F32 else 0x7fff
    y = voxq.lora(x, a, b, cu, ints([0, 1]), scale, base=base)
    want[:rows[0]] = True
    assert torch.equal(torch.isnan(y), want)


@pytest.mark.parametrize("dt,wt", LORA_TYPES, ids=ids)
@pytest.mark.parametrize("rank", [8, 24, 40, 72])
@pytest.mark.parametrize("rows", [[5, 3, 1, 4], [4000, 900, 3, 700]], ids=["few", "many"])
def test_lora_that_meets_infinities_and_nan(rows, rank, dt, wt):
    """Infinite and NaN inputs, weights and hidden values give what the formula gives, and harm no other row or column."""
    K, N = 264, 520
    x, a, b, cu, _, scale, base = lora_inputs(rows, 4, K, N, rank, dt, wt, seed=9)
    who, ranks = ints([0, 1, 2, 3]), ints([rank, rank - 3, rank, rank])
    inf, nan = float("inf"), float("nan")
    top = torch.finfo(dt).max
    a[0, :, 5], b[0, :40] = a[0, :, 5].abs() + 0.01, b[0, :40].abs() + 0.01
    a[0, :, 11] = 2e-38 if wt is F32 else 0       # beside a value next to the type's end: a small product, or nothing
    x[0, 11], x[1, 5], x[2, 5], x[3, 7], x[4, 100] = top, inf, -inf, nan, inf
    b[1, 9, 1], b[1, 10, 0], b[1, 300, 2] = inf, -inf, nan
    a[1, rank - 3:], b[1, :, rank - 3:] = nan, inf   # past the adapter's own rank
    a[2, 3, 9] = inf
    base[rows[0], 17] = inf
    bound_of = [torch.nan_to_num(t, 0, 0, 0) for t in (x, a, b, base)]
    _, bound = R.adapters(bound_of[0], bound_of[1], bound_of[2], cu, who, scale, bound_of[3], ranks)
    y = R.f8(voxq.lora(x, a, b, cu, who, scale, base=base, ranks=ranks))
    ref = R.f8(base).clone()
    for s, r in enumerate(ranks.tolist()):
        at = slice(int(cu[s]), int(cu[s + 1]))
        ref[at] += float(scale[s]) * (R.f8(x[at]) @ R.f8(a[s, :r]).T @ R.f8(b[s, :, :r]).T)
    at = torch.zeros_like(ref, dtype=torch.bool)  # an infinity in B may come out as a NaN
    at[rows[0]:rows[0] + rows[1], 9:11] = True
    assert not torch.isfinite(ref[at]).any()
    ref[at & torch.isnan(y)] = nan
    assert torch.equal(torch.isnan(y), torch.isnan(ref)), "NaN in other places than the formula's"
    fine = torch.isfinite(ref)
    assert torch.equal(y[~fine & ~torch.isnan(ref)], ref[~fine & ~torch.isnan(ref)]), "infinities in other places than the formula's"
    R.assert_within(torch.where(fine, y, 0.0), torch.where(fine, ref, 0.0), bound)
