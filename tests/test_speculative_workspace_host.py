"""The workspace of draft verification covers every call that it may serve: the
same sizes in greedy decoding, which leaves the draft logits out, and smaller
batches and shorter drafts, whose rows are cut into shorter chunks."""

from __future__ import annotations

import pytest

from rosellm_amd import _native as nat


@pytest.fixture(scope="module")
def size():
    if not nat.LIB_PATH.exists():
        pytest.skip("librosellm_amd.so is not built (run __graft_entry__.build())")
    return nat.load().rrl_verify_drafts_workspace_bytes


def _need(rows, B, V):
    """Statistics (16 bytes a chunk, and a row), masses and plans of a call of B sequences and `rows` rows."""
    least = rows * -(-V // 1024)
    chunk = 1024 if least <= 16384 else (2048 if least <= 40960 else 4096)
    return 16 * rows * -(-V // chunk) + 16 * rows + 8 * B * -(-V // 1024) + 8 * B


# vocabularies of up to 17 million entries, the last with more chunks to a row than the borders
@pytest.mark.parametrize("V", [1, 1000, 4096, 4097, 32000, 50257, 151936, 262144, 17_000_000])
def test_verify_workspace_covers_smaller_calls(size, V):
    for K in (0, 1, 2, 4, 5, 8, 13):
        last = 0
        for B in range(1, 260):
            with_draft, without = size(B, K, V, 1), size(B, K, V, 0)
            if with_draft == 0:  # refused
                assert B * (2 * K + 1) * -(-V // 4096) > 1 << 23
                break
            assert with_draft >= without, (B, K, V)
            assert with_draft >= _need(B * (2 * K + 1), B, V) and without >= _need(B * (K + 1), B, V), (B, K, V)
            assert without >= last, (B, K, V)
            last = without
            if K > 0:
                assert with_draft >= size(B, K - 1, V, 1), (B, K, V)
            if B > 1:
                assert with_draft >= size(B - 1, K, V, 1), (B, K, V)
