"""How long a row tokens are drawn from may be, which the C entry point checks before any launch."""

from __future__ import annotations

import pytest

from rosellm_amd import _native as nat


def test_rows_whose_sums_are_too_coarse_are_refused():
    """A sum's worst error, V half units of 2^-44 (2^-(62 - b) past 2^18 entries) of the
    largest weight, stays within 2^-23 of it."""
    if not nat.LIB_PATH.exists():
        pytest.skip("librosellm_amd.so is not built (run __graft_entry__.build())")
    lib = nat.load()
    size = lib.rrl_sample_tokens_workspace_bytes

    def error(V):
        bits = (V - 1).bit_length()
        return V * 2.0 ** -(62 - bits if bits > 18 else 44) / 2

    for V in (1, 151936, 1 << 18, 300001, 1 << 20, (1 << 20) + 1, 1 << 21, 1 << 30):
        fits = error(V) <= 2.0 ** -23
        assert (size(1, V, None) > 0) == fits, V
        if not fits:
            p = nat.RrlSampleParams(1.0, 1.0, 0.0, 0, None, None, None, None, nat.I32)
            assert lib.rrl_sample_tokens(16, nat.BF16, 1, V, V, 16, p, 16, 16, None, 16, None) == -1
            assert b"2^20 entries" in lib.rrl_last_error()
