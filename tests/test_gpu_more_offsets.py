"""Operands past 2^32 elements: sampling from given uniforms, adapters and dropout (MI355X)."""

from __future__ import annotations

import pytest
import torch

from rosellm_amd.roseinfer import sample_tokens
from rosellm_amd.rosetrainer import adapter_linear, dropout

from _philox import philox

pytestmark = [pytest.mark.gpu, pytest.mark.slow]


@pytest.fixture(autouse=True)
def _release():
    yield
    torch.cuda.empty_cache()


def test_sample_rows_far_apart(device):
    big = torch.zeros(3, (1 << 31) + 64, dtype=torch.bfloat16, device=device)
    small = (torch.randn(3, 5000, device=device) * 3).bfloat16()
    big[:, :5000] = small
    u = torch.rand(3, device=device)
    for kw in (dict(), dict(top_k=40, top_p=0.8), dict(top_p=0.9)):
        for a, b in zip(sample_tokens(big[:, :5000], u, **kw), sample_tokens(small, u, **kw)):
            assert torch.equal(a, b)


def test_adapter_rows_far_apart(device):
    big = torch.zeros(3, (1 << 31) + 64, dtype=torch.bfloat16, device=device)
    x, base = torch.randn(3, 64, device=device).bfloat16(), torch.randn(3, 48, device=device).bfloat16()
    big[:, :64], big[:, 100:148] = x, base
    down, up = torch.randn(2, 8, 64, device=device).bfloat16(), torch.randn(2, 48, 8, device=device).bfloat16()
    ids = torch.tensor([1, -1, 0], device=device)
    got = adapter_linear(big[:, :64], down, up, ids, base=big[:, 100:148])
    assert torch.equal(got, adapter_linear(x, down, up, ids, base=base))


def test_many_adapter_rows(device):
    """Rows whose product and input lie past 2^32 elements: the last ones against a call on them alone."""
    N, H = (1 << 22) + 1500, 1032
    x = torch.zeros(N, H, dtype=torch.bfloat16, device=device)
    x[-1500:].normal_()
    down, up = torch.randn(1, 16, H, device=device).bfloat16(), torch.randn(1, H, 16, device=device).bfloat16()
    y = adapter_linear(x, down, up)
    assert not y[:1000].any()
    assert torch.equal(y[-1500:], adapter_linear(x[-1500:], down, up))


def test_dropout_of_many_entries(device):
    n = (1 << 32) + 4096
    x = torch.ones(n, dtype=torch.bfloat16, device=device)
    y = dropout(x, 0.5, seed=3, offset=1)
    for at in (0, (1 << 32) - 64, n - 64):
        import numpy as np

        i = np.arange(at // 8, at // 8 + 8, dtype=np.uint64)
        words = philox(np.stack([i & np.uint64(0xFFFFFFFF), i >> np.uint64(32), np.full_like(i, 1), np.zeros_like(i)], -1), 3)
        halves = np.stack([words & np.uint64(0xFFFF), words >> np.uint64(16)], -1).reshape(-1)
        assert torch.equal(y[at:at + 64].cpu() != 0, torch.from_numpy(halves >= np.uint64(32768)))
