"""Host side of the batched step where its arguments meet their limits: refusals before any launch."""
from __future__ import annotations

import ctypes as C
import importlib.util
import os
import subprocess
import sys

import pytest

torch = pytest.importorskip("torch")
import voxq  # noqa: E402
from test_batched_cpu import P, REPO, norm, rope  # noqa: E402


@pytest.mark.parametrize("off", [1, 2, 4, 12])
def test_rotary_tables_between_pairs_are_refused(off):
    """(cos, sin) pairs are read and written in one access: a table that starts inside one would fault on the device."""
    L = voxq.lib()
    assert L.voxq_rope_append(C.byref(rope(freqs=P + off)), None) == voxq.UNSUPPORTED
    d = voxq.RopeTableDesc(n_pos=4, rot_dim=8, theta=1e4, out=P + off)
    assert L.voxq_rope_freqs(C.byref(d), None) == voxq.UNSUPPORTED


def test_norm_rows_between_elements_are_refused():
    L = voxq.lib()
    for kw in (dict(y=P + 1), dict(x=P + 2), dict(n_out=P + 3), dict(w_pre=P + 2), dict(w_post=P + 1), dict(gate=P + 2, gate_rows=1, ldg=64)):
        assert L.voxq_norm_residual(C.byref(norm(**kw)), None) == voxq.UNSUPPORTED, kw
    assert L.voxq_norm_residual(C.byref(norm(dtype=voxq.F16, h_out=P + 1)), None) == voxq.UNSUPPORTED


def test_shared_memory_is_asked_for_on_every_device(tmp_path):
    """allow_shared against a stand-in runtime: once a device, again after a failure."""
    src = tmp_path / "t.cpp"
    src.write_text(r'''
#include "voxq_internal.h"
static int dev, calls, fail;
extern "C" cudaError_t cudaGetDevice(int* d) { *d = dev; return cudaSuccess; }
extern "C" cudaError_t cudaFuncSetAttribute(const void*, cudaFuncAttribute, int) {
    calls++;
    return fail ? cudaErrorInvalidValue : cudaSuccess;
}
int main() {
    std::atomic<uint64_t> asked{0};
    auto ask = [&](int d, int f) { dev = d; fail = f; return voxq::allow_shared(nullptr, 100000, asked); };
    if (ask(0, 1) == cudaSuccess || calls != 1) return 1;
    if (ask(0, 0) != cudaSuccess || calls != 2) return 2;
    if (ask(0, 1) != cudaSuccess || calls != 2) return 3;
    if (ask(1, 0) != cudaSuccess || calls != 3) return 4;
    if (ask(63, 0) != cudaSuccess || ask(63, 1) != cudaSuccess || calls != 4) return 5;
    if (ask(64, 0) != cudaSuccess || ask(64, 0) != cudaSuccess || calls != 6) return 6;
    return 0;
}
''')
    exe = tmp_path / "t"
    cuda = os.path.join(os.path.dirname(os.path.dirname(os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc"))), "include")
    subprocess.run(["g++", "-std=c++17", "-I", os.path.join(REPO, "include"), "-I", os.path.join(REPO, "voxcpm2-c_b200", "csrc"), "-I", cuda,
                    str(src), "-o", str(exe)], check=True)
    assert subprocess.run([str(exe)]).returncode == 0


def test_tensors_of_several_gpus_are_refused():
    """Each call with one of its tensors on a second GPU, the others on the first (fake tensors: shapes and devices without
    memory, so nothing can be launched)."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    i32, i64 = torch.int32, torch.int64
    calls = {
        voxq.paged_attention: [((1, 4, 64),), ((2, 16, 2, 64),), ((2, 16, 2, 64),), ((1, 2), i32), ((2,), i32), ((1,), i32), 1, 16, True, 0.0, ((1, 4, 64),)],
        voxq.rope_append: [((1, 4, 64),), ((1, 2, 64),), ((1, 2, 64),), ((8, 32, 2),), ((1,), i32), ((1,), i64), ((2, 16, 2, 64),), ((2, 16, 2, 64),), ((1, 4, 64),)],
        voxq.lora: [((2, 64),), ((1, 8, 64),), ((1, 32, 8),), ((2,), i32), ((1,), i32), ((1,),), ((2, 32),), ((2, 32),), ((1,), i32)],
        voxq.norm_residual: [((2, 64),), ((2, 64),), ((64,),), ((64,),), ((3, 64),), ((2,), i32), 1.0, 1e-5, ((2, 64),), ((2, 64),)],
    }
    with FakeTensorMode():
        for f, spec in calls.items():
            for away in [i for i, s in enumerate(spec) if isinstance(s, tuple)]:
                args = [s if not isinstance(s, tuple) else
                        torch.empty(s[0], dtype=s[1] if len(s) > 1 else torch.float32, device=f"cuda:{int(i == away)}") for i, s in enumerate(spec)]
                with pytest.raises(ValueError, match="one GPU"):
                    f(*args)


def test_streams_of_another_gpu_are_refused():
    from torch._subclasses.fake_tensor import FakeTensorMode

    class Stream:
        cuda_stream, device = 0, torch.device("cuda:1")

    with FakeTensorMode():
        y = torch.empty(2, 64, device="cuda:0")
        with pytest.raises(ValueError, match="stream"):
            voxq.norm_residual(y, y, stream=Stream())
    with pytest.raises(ValueError):
        voxq.norm_residual(torch.zeros(2, 64), torch.zeros(2, 64), stream=Stream())


def _build_module(tmp_path, monkeypatch):
    spec = importlib.util.spec_from_file_location("voxq_build", os.path.join(REPO, "voxcpm2-c_b200", "build.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    (tmp_path / "voxq").mkdir()
    monkeypatch.setattr(m, "HERE", str(tmp_path))
    monkeypatch.setattr(m, "OBJ", str(tmp_path / "_build"))
    ran = []

    def compiled(cmd, **kw):
        ran.append(cmd)
        (tmp_path / "voxq" / "_torch.so").write_text("")
        return subprocess.CompletedProcess(cmd, 0, "", "")
    monkeypatch.setattr(m.subprocess, "run", compiled)
    return m, ran


def test_the_library_builds_without_pytorch(tmp_path, monkeypatch):
    m, ran = _build_module(tmp_path, monkeypatch)
    monkeypatch.setitem(sys.modules, "torch", None)  # its import then fails
    assert m.build_binding() is None and not ran


def test_the_binding_is_rebuilt_for_another_torch(tmp_path, monkeypatch):
    m, ran = _build_module(tmp_path, monkeypatch)
    assert m.build_binding() and len(ran) == 1
    assert m.build_binding() and len(ran) == 1
    monkeypatch.setattr(torch, "__version__", "0.0.another")
    assert m.build_binding() and len(ran) == 2


def test_an_output_of_another_type_than_asked_for_is_refused():
    z = torch.zeros
    with pytest.raises(ValueError, match="differ"):
        voxq.paged_attention(z(1, 4, 64), z(2, 16, 2, 64), z(2, 16, 2, 64), None, None, None, 1, 16, out=z(1, 4, 64), out_dtype=torch.float16)
