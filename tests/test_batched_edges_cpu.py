"""Host side of the batched step where its arguments meet their limits: refusals before any launch."""
from __future__ import annotations

import ctypes as C

import pytest

torch = pytest.importorskip("torch")
import voxq  # noqa: E402
from test_batched_cpu import P, norm, rope  # noqa: E402


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
