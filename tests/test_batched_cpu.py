"""Host side of the batched step: the descriptors' layout, the calls' refusals before any launch, and the paged
cache's bookkeeping."""
from __future__ import annotations

import ctypes as C
import os
import random
import subprocess

import pytest

torch = pytest.importorskip("torch")
import voxq  # noqa: E402
from voxq.batched_block import BatchedBlock, PagedCache  # noqa: E402

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
DESCS = {"voxq_rope_table": voxq.RopeTableDesc, "voxq_rope": voxq.RopeDesc, "voxq_paged_attn": voxq.PagedAttnDesc,
         "voxq_lora": voxq.LoraDesc, "voxq_norm": voxq.NormDesc}


def test_descriptor_layouts_match_the_header(tmp_path):
    """Every field's offset, and what the packed form writes, against the C compiler's view of voxq.h."""
    lines = []
    for name, cls in DESCS.items():
        lines.append(f'printf("{name} %zu", sizeof({name}));')
        lines += [f'printf(" %zu", offsetof({name}, {f}));' for f, _ in cls._fields_]
        lines.append('printf("\\n");')
    src = tmp_path / "layout.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include <stdbool.h>\n#include "voxq.h"\nint main(void) {\n' +
                   "\n".join(lines) + "\nreturn 0; }\n")
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-I", os.path.join(REPO, "include"), str(src), "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout
    for line in out.splitlines():
        name, size, *offs = line.split()
        cls = DESCS[name]
        assert C.sizeof(cls) == int(size)
        assert [getattr(cls, f).offset for f, _ in cls._fields_] == [int(o) for o in offs], name
        if hasattr(cls, "pack"):
            vals = [float(i % 100) if t in (C.c_float, C.c_double) else i + 1 for i, (_, t) in enumerate(cls._fields_)]
            raw = cls.pack(*vals)
            assert len(raw) == int(size)
            d = cls.from_buffer_copy(raw)
            assert [getattr(d, f) for f, _ in cls._fields_] == vals, name


P = 1 << 20  # an aligned address that no call gets as far as using


def attn(**kw):
    d = dict(q=P, q_stride=1024, q_head_stride=64, out=P, o_stride=1024, o_head_stride=64, k=P, v=P, page_stride=2048,
             row_stride=128, head_stride=64, block_table=P, table_stride=8, cu_q=P, kv_len=P, batch=1, heads=16, kv_heads=2,
             head_dim=64, pages=9, page_size=16, total_q=1, max_q=1, max_kv=100, dtype=voxq.BF16, out_dtype=voxq.BF16, causal=1)
    return voxq.PagedAttnDesc(**{**d, **kw})


def rope(**kw):
    d = dict(q=P, k=P, v=P, q_stride=1024, q_head_stride=64, k_stride=128, k_head_stride=64, v_stride=128, v_head_stride=64,
             q_out=P, qo_stride=1024, qo_head_stride=64, cache_k=P, cache_v=P, page_stride=2048, row_stride=128, head_stride=64,
             freqs=P, positions=P, slots=P, tokens=1, heads=16, kv_heads=2, head_dim=64, rot_dim=64, n_pos=10, pages=9,
             page_size=16, in_dtype=voxq.F32, cache_dtype=voxq.BF16)
    return voxq.RopeDesc(**{**d, **kw})


def lora(**kw):
    d = dict(x=P, ldx=64, base=P, ldb=64, out=P, ldo=64, a=P, b=P, cu=P, adapter=P, ranks=0, scale=P, rows=1, batch=1, K=64,
             N=64, rank=8, adapters=1, dtype=voxq.F32, w_dtype=voxq.BF16)
    return voxq.LoraDesc(**{**d, **kw})


def norm(**kw):
    d = dict(y=P, x=P, ldy=64, ldx=64, w_pre=P, h_out=P, n_out=P, ldh=64, ldn=64, rows=1, D=64, dtype=voxq.F32, alpha=1, eps=1e-5)
    return voxq.NormDesc(**{**d, **kw})


BAD_SHAPE, BAD_KIND, BAD_NULL = voxq.SHAPE_MISMATCH, voxq.UNSUPPORTED, voxq.INTERNAL
REFUSED = [
    ("voxq_paged_attention", attn, [
        (dict(heads=15), BAD_SHAPE), (dict(batch=0), BAD_SHAPE), (dict(total_q=-1), BAD_SHAPE), (dict(max_kv=129), BAD_SHAPE),
        (dict(page_size=0), BAD_SHAPE), (dict(kv_heads=0), BAD_SHAPE), (dict(pages=0), BAD_SHAPE), (dict(dtype=voxq.Q4), BAD_KIND),
        (dict(out_dtype=voxq.F16), BAD_KIND), (dict(head_dim=68), BAD_KIND), (dict(head_dim=264), BAD_KIND),
        (dict(q=P + 8), BAD_KIND), (dict(row_stride=100), BAD_KIND), (dict(o_stride=1025), BAD_KIND), (dict(v=P + 2), BAD_KIND),
        (dict(total_q=1 << 28), BAD_KIND), (dict(q=0), BAD_NULL), (dict(block_table=0), BAD_NULL), (dict(kv_len=0), BAD_NULL)]),
    ("voxq_rope_append", rope, [
        (dict(rot_dim=66), BAD_SHAPE), (dict(rot_dim=7), BAD_SHAPE), (dict(tokens=-1), BAD_SHAPE), (dict(n_pos=0), BAD_SHAPE),
        (dict(in_dtype=voxq.F16), BAD_KIND), (dict(cache_dtype=7), BAD_KIND), (dict(head_dim=60, rot_dim=60), BAD_KIND),
        (dict(q=P + 4), BAD_KIND), (dict(cache_v=P + 2), BAD_KIND), (dict(k_stride=130), BAD_KIND),
        (dict(pages=1 << 20, page_size=1 << 12), BAD_KIND), (dict(k=0), BAD_NULL), (dict(positions=0), BAD_NULL),
        (dict(slots=0), BAD_NULL), (dict(freqs=0), BAD_NULL)]),
    ("voxq_lora_forward", lora, [
        (dict(rows=-1), BAD_SHAPE), (dict(batch=0), BAD_SHAPE), (dict(K=60), BAD_KIND), (dict(N=63), BAD_KIND), (dict(rank=12), BAD_KIND),
        (dict(rank=136), BAD_KIND), (dict(dtype=voxq.F16), BAD_KIND), (dict(w_dtype=voxq.Q8), BAD_KIND), (dict(ldx=65), BAD_KIND),
        (dict(base=P + 4), BAD_KIND), (dict(out=0), BAD_NULL), (dict(scale=0), BAD_NULL), (dict(cu=0), BAD_NULL)]),
    ("voxq_norm_residual", norm, [
        (dict(rows=-1), BAD_SHAPE), (dict(gate=P, gate_rows=0), BAD_SHAPE), (dict(gate=P, gate_rows=3), BAD_SHAPE),
        (dict(D=16385), BAD_KIND), (dict(dtype=9), BAD_KIND), (dict(y=0), BAD_NULL), (dict(w_pre=0), BAD_NULL),
        (dict(h_out=0, n_out=0), BAD_NULL)]),
]


@pytest.mark.parametrize("name,make,cases", REFUSED, ids=[r[0] for r in REFUSED])
def test_refusals(name, make, cases):
    f = getattr(voxq.lib(), name)
    for kw, code in cases:
        assert f(C.byref(make(**kw)), None) == code, f"{name} {kw}"
    assert f(None, None) == BAD_NULL


def test_nothing_to_do_succeeds_without_a_device():
    L = voxq.lib()
    assert L.voxq_paged_attention(C.byref(attn(total_q=0)), None) == 0
    assert L.voxq_rope_append(C.byref(rope(tokens=0)), None) == 0
    assert L.voxq_lora_forward(C.byref(lora(rows=0)), None) == 0
    assert L.voxq_norm_residual(C.byref(norm(rows=0)), None) == 0
    for kw, code in ((dict(rot_dim=3), BAD_SHAPE), (dict(theta=1.0), BAD_SHAPE), (dict(scaling=9), BAD_KIND), (dict(rot_dim=512), BAD_KIND),
                     (dict(scaling=1, factor=0.0), BAD_SHAPE), (dict(scaling=2, factor=2.0, rot_dim=2), BAD_SHAPE),
                     (dict(scaling=3, factor=2.0), BAD_SHAPE), (dict(scaling=4), BAD_NULL), (dict(out=0), BAD_NULL)):
        d = voxq.RopeTableDesc(**{**dict(n_pos=4, rot_dim=8, theta=1e4, out=P), **kw})
        assert L.voxq_rope_freqs(C.byref(d), None) == code, kw


def test_workspace_is_asked_for_when_keys_are_split():
    L = voxq.lib()
    ask = lambda **kw: L.voxq_paged_attention_workspace(C.byref(attn(**kw)))  # noqa: E731
    assert ask(total_q=0) == 0 and ask(max_kv=129) == 0
    need = ask(max_kv=30000, table_stride=1875)
    assert need > 0 and need % 4 == 0
    d = attn(max_kv=30000, table_stride=1875)
    assert L.voxq_paged_attention(C.byref(d), None) == BAD_NULL
    d.workspace, d.workspace_bytes = P, need - 1
    assert L.voxq_paged_attention(C.byref(d), None) == voxq.OOM
    d.workspace, d.workspace_bytes = P + 16, need
    assert L.voxq_paged_attention(C.byref(d), None) == BAD_KIND


def test_paged_cache_places():
    """Random steps: no two live positions share a place, tables and slots agree, pages come back."""
    rng = random.Random(3)
    c = PagedCache(1, 40, 4, 1, 8, dtype=torch.float32, device="cpu")
    place = {}
    for _ in range(60):
        live = rng.sample("abcdefgh", rng.randint(1, 5))
        ask = [(s, rng.randint(0, 9)) for s in live]
        before = {s: c.length(s) for s in live}
        if sum(max(0, -(-(before[s] + n) // 4) - -(-before[s] // 4)) for s, n in ask) > c.free_pages:
            free = c.free_pages
            with pytest.raises(MemoryError):
                c.step(ask)
            assert c.free_pages == free and all(c.length(s) == before[s] for s in live)
            gone = rng.choice([s for s in "abcdefgh" if c.length(s)])
            c.release(gone)
            place.pop(gone, None)
            continue
        st = c.step(ask, adapters={"a": 2})
        assert st.tokens == sum(n for _, n in ask) and st.max_q == max(n for _, n in ask)
        for i, (s, n) in enumerate(ask):
            lo, hi = int(st.cu[i]), int(st.cu[i + 1])
            assert hi - lo == n and int(st.kv_len[i]) == before[s] + n and int(st.adapter[i]) == (2 if s == "a" else -1)
            assert st.positions[lo:hi].tolist() == list(range(before[s], before[s] + n))
            place.setdefault(s, []).extend(st.slots[lo:hi].tolist())
            assert place[s] == [int(st.table[i, j // 4]) * 4 + j % 4 for j in range(before[s] + n)]
        used = [x for v in place.values() for x in v]
        assert len(set(used)) == len(used) and all(x >= 4 for x in used)
    for s in "abcdefgh":
        c.release(s)
    assert c.free_pages == 39
    with pytest.raises(ValueError):
        c.step([("a", 1), ("a", 2)])
    with pytest.raises(ValueError):
        PagedCache(1, 1, 4, 1, 8, device="cpu")


def test_block_refuses_adapters_beside_the_fused_pair():
    with pytest.raises(ValueError):
        BatchedBlock(*[None] * 9, heads=1, kv_heads=1, adapters={"w1": None})


def test_binding_refuses_host_tensors_and_other_objects():
    z = torch.zeros
    ints = z(2, dtype=torch.int32)
    cache = z(2, 16, 2, 64)
    for f, args in ((voxq.paged_attention, (z(1, 4, 64), cache, cache, z(1, 2, dtype=torch.int32), ints, ints[:1], 1, 16)),
                    (voxq.rope_append, (z(1, 4, 64), z(1, 2, 64), z(1, 2, 64), None, None, z(1, dtype=torch.int64), cache, cache)),
                    (voxq.lora, (z(2, 64), z(1, 8, 64), z(1, 32, 8), ints, ints[:1], z(1))),
                    (voxq.norm_residual, (z(2, 64), z(2, 64)))):
        with pytest.raises(ValueError):
            f(*args)
        with pytest.raises(ValueError):
            f(None, *args[1:])
        with pytest.raises(ValueError):
            f([1.0], *args[1:])
