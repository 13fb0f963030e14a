"""The product's C entry point refuses scales at an address that its loads of four do not allow."""

from __future__ import annotations

import pytest

from rosellm_amd import _native as nat


@pytest.mark.parametrize("scales", [17, 18, 19])
def test_mxfp4_linear_refuses_misaligned_scales(scales):
    if not nat.LIB_PATH.exists():
        pytest.skip("librosellm_amd.so is not built (run __graft_entry__.build())")
    lib = nat.load()
    rc = lib.rrl_mxfp4_linear(16, nat.BF16, 2, 64, 64, 16, scales, 3, 16, nat.F32, 16, None)
    assert rc == -4 and b"scales: 4" in lib.rrl_last_error()
