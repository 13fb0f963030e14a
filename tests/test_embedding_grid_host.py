"""The gradient's size check counts the workgroups that are launched: 16-bit rows that
allow 8-byte accesses are read by 4 bytes, twice as many columns' shares as 8-byte ones
would make.  (Refused before any launch, so the addresses are never used.)"""

from __future__ import annotations

import pytest

from rosellm_amd import _native as nat


@pytest.mark.parametrize("dtype", [nat.BF16, nat.F16])
def test_embedding_gradient_refuses_grids_past_32_bits(dtype):
    if not nat.LIB_PATH.exists():
        pytest.skip("librosellm_amd.so is not built (run __graft_entry__.build())")
    lib = nat.load()
    # 2.97 million pieces of 64 positions x 9 shares of 128 columns, in workgroups of 256 threads
    assert 190_000_000 // 64 * 9 * 256 >= 1 << 32
    rc = lib.rrl_embedding_bwd(16, nat.I64, 190_000_000, 16, dtype, 1000, 1028, 1028, 1.0, 0, 0, 16, 1028, 16, None)
    assert rc == -1 and b"too many ids or rows" in lib.rrl_last_error()
