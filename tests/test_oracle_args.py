"""The CPU checker's own arguments."""
from __future__ import annotations

import numpy as np
import pytest

from oracle import oracle as O


def test_matmul_nt_takes_only_an_output_that_fits():
    """`out` goes to C as a pointer: another type, shape or layout, or memory that is not to be written, is refused."""
    a, w = np.ones((3, 8), np.float32), np.ones((5, 8), np.float32)
    fixed = np.zeros((3, 5), np.float32)
    fixed.flags.writeable = False
    for bad in (np.zeros((3, 5)), np.zeros((5, 5), np.float32), np.zeros(15, np.float32), np.zeros((3, 10), np.float32)[:, ::2], fixed):
        with pytest.raises(ValueError):
            O.matmul_nt(a, w, out=bad)
    out = np.full((3, 5), 7, np.float32)
    assert O.matmul_nt(a, w, out=out) is out and (out == 8).all()
