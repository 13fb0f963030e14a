"""A scale that float32 does not hold is refused: as an infinity it would turn zeros into NaN."""

from __future__ import annotations

import pytest
import torch

from rosellm_amd import _native as nat
from rosellm_amd.rosetrainer import embedding

# the first number that rounds to infinity is half a step (2^103) past the largest
LARGEST = float(torch.finfo(torch.float32).max)
PAST = [LARGEST + 2.0 ** 103, 1e39, -1e300]


def test_embedding_refuses_a_scale_past_float32():
    ids, w = torch.zeros(3, dtype=torch.long), torch.zeros(4, 8)
    for scale in PAST:
        with pytest.raises(ValueError, match="float32's range"):
            embedding(ids, w, scale=scale)
    for scale in (LARGEST, LARGEST + 2.0 ** 102, 1e-300, float("inf"), float("nan")):
        with pytest.raises(RuntimeError, match="ROCm GPU"):  # past the argument checks
            embedding(ids, w, scale=scale)


def test_embedding_entry_points_refuse_a_scale_past_float32():
    if not nat.LIB_PATH.exists():
        pytest.skip("librosellm_amd.so is not built (run __graft_entry__.build())")
    lib = nat.load()
    for scale in PAST:
        assert lib.rrl_embedding_fwd(16, nat.I64, 2, 16, nat.F32, 4, 8, 8, scale, 0, 0, 16, None) == -1
        assert b"float32's range" in lib.rrl_last_error()
        assert lib.rrl_embedding_bwd(16, nat.I64, 2, 16, nat.F32, 4, 8, 8, scale, 0, 0, 16, 8, 16, None) == -1
        assert b"float32's range" in lib.rrl_last_error()
    for scale in (LARGEST, float("inf"), float("nan")):
        assert lib.rrl_embedding_fwd(16, nat.I64, 0, 16, nat.F32, 4, 8, 8, scale, 0, 0, 16, None) == 0
