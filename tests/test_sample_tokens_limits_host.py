"""How long a row tokens are drawn from may be, which the C entry point checks before any
launch, and the workspace that it asks for."""

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


@pytest.mark.parametrize("B", [1, 4, 200])
@pytest.mark.parametrize("V", [1, 9, 64, 65, 1000, 4095, 4096, 8192, 8193, 50257, 151936])
def test_workspace(B, V):
    """What a cut takes beside the rest: bins of sums (8 bytes) for a top-p, of counts (4) with
    a maximum of each of 256 lanes (4) and a list of a row's entries (8) for a top-k."""
    if not nat.LIB_PATH.exists():
        pytest.skip("librosellm_amd.so is not built (run __graft_entry__.build())")
    size = nat.load().rrl_sample_tokens_workspace_bytes
    part = 8192  # entries, twice as many where a thousand workgroups are left
    while part < 65536 and B * -(-V // (2 * part)) >= 1024:
        part *= 2
    parts = B * -(-V // part)
    bins = min(1024, max(64, 1 << (V - 1).bit_length()))
    top_p = 8 * bins * parts
    top_k = 4 * bins * parts + 4 * 256 * parts + 8 * B * min(V, 4096)
    of = lambda k, p: size(B, V, nat.RrlSampleParams(1.0, p, 0.0, k))
    none = of(0, 1.0)
    small = 256 * 8  # each piece starts at a multiple of 256, and a few are a number or two a row
    assert none >= parts * (4 + 8 + 4 * 8 + 2 * 4 * 16) + 8 * B
    assert top_p <= of(0, 0.5) - none <= top_p + small
    if V > 1:  # (no top-k leaves out anything of one entry)
        assert top_k <= of(1, 1.0) - none <= top_k + 8 * B + small
        assert top_k + top_p <= of(1, 0.5) - none <= top_k + top_p + 8 * B + small
        assert of(1, 0.5) == size(B, V, None)


def test_workspace_of_many_short_rows():
    if not nat.LIB_PATH.exists():
        pytest.skip("librosellm_amd.so is not built (run __graft_entry__.build())")
    assert nat.load().rrl_sample_tokens_workspace_bytes(131072, 9, None) < 1 << 29
