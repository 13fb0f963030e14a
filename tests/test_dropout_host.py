"""Dropout's argument checks, which run before any tensor reaches a device, its mask's
definition, and the C entry point's host-side validation."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

from rosellm_amd import _native as nat
from rosellm_amd.rosetrainer import dropout

from _philox import philox


def test_dropout_refusals():
    x = torch.zeros(3, 8)
    with pytest.raises(TypeError, match="float32, bfloat16 or float16"):
        dropout(x.double(), 0.1)
    for p in (-0.1, 1.1, float("nan")):
        with pytest.raises(ValueError, match="in \\[0, 1\\]"):
            dropout(x, p)
    with pytest.raises(ValueError, match="residual must have shape"):
        dropout(x, 0.1, residual=torch.zeros(8))
    with pytest.raises(TypeError, match="residual must have the dtype"):
        dropout(x, 0.1, residual=torch.zeros(3, 8, dtype=torch.bfloat16))
    with pytest.raises(TypeError, match="offset"):
        dropout(x, 0.1, offset=torch.zeros(2, dtype=torch.int64))
    with pytest.raises(TypeError, match="offset"):
        dropout(x, 0.1, offset=torch.zeros(1, dtype=torch.int32))
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        dropout(x, 0.1)


@pytest.fixture(scope="module")
def lib():
    if not nat.LIB_PATH.exists():
        pytest.skip("librosellm_amd.so is not built (run __graft_entry__.build())")
    return nat.load()


def test_the_tests_generator_is_the_librarys(lib):
    rng = np.random.default_rng(0)
    for _ in range(50):
        c = rng.integers(0, 2 ** 32, 4, dtype=np.uint64)
        seed = int(rng.integers(0, 2 ** 63, dtype=np.uint64)) * 2 + 1
        got = (ctypes.c_uint32 * 4)(*(int(v) for v in c))
        lib.rrl_philox4x32_10(got, (ctypes.c_uint32 * 2)(seed & 0xFFFFFFFF, seed >> 32))
        assert [int(v) for v in philox(c[None], seed)[0]] == list(got)


def test_entry_point_validation(lib):
    def call(x=16, dt=nat.BF16, rows=2, cols=8, ld=8, res=None, rld=0, p=0.1, at=None, out=16):
        return lib.rrl_dropout(x, dt, rows, cols, ld, res, rld, nat.RrlDropoutParams(p, 1, 2, at), out, None)

    assert call(rows=0) == 0 and call(cols=0) == 0
    assert call(dt=nat.F64) == -2 and b"float32" in lib.rrl_last_error()
    assert call(rows=-1) == -1 and b"negative" in lib.rrl_last_error()
    assert call(p=-0.5) == -1 and b"probability" in lib.rrl_last_error()
    assert call(p=float("nan")) == -1 and call(p=1.5) == -1
    assert call(x=None) == -1 and call(out=None) == -1 and b"null" in lib.rrl_last_error()
    assert lib.rrl_dropout(16, nat.BF16, 2, 8, 8, None, 0, None, 16, None) == -1
    assert call(ld=-8) == -1 and call(res=16, rld=-1) == -1
    assert call(rows=1 << 32) == -1 and b"2^32" in lib.rrl_last_error()
    assert call(rows=1, cols=1 << 36) == -1
    assert call(x=17) == -4 and call(out=17) == -4 and call(res=17) == -4 and call(at=12) == -4
    assert b"aligned" in lib.rrl_last_error()
