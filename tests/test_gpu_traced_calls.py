"""Calls that torch.jit.trace records, run again on other inputs (MI355X)."""

from __future__ import annotations

import pytest
import torch

from rosellm_amd.rosetrainer import adapter_linear, dropout

pytestmark = pytest.mark.gpu


def _trace(f, *args):
    return torch.jit.trace(f, args, check_trace=False)


def test_dropout(device):
    x, r = torch.randn(2, 40, 64, device=device), torch.randn(2, 40, 64, device=device)
    f = _trace(lambda a, b: dropout(a, 0.3, seed=5, residual=b) * 2, x[0], r[0])
    for k in (1, 0, 1):
        assert torch.equal(f(x[k], r[k]), dropout(x[k], 0.3, seed=5, residual=r[k]) * 2)
    at = torch.zeros(1, dtype=torch.int64, device=device)
    f = _trace(lambda a, o: dropout(a, 0.3, seed=5, offset=o), x[0], at)
    for k in (0, 3):
        assert torch.equal(f(x[1], at + k), dropout(x[1], 0.3, seed=5, offset=k))


def test_adapters(device):
    gen = torch.Generator().manual_seed(1)
    x, base = torch.randn(2, 30, 48, generator=gen).to(device), torch.randn(2, 30, 56, generator=gen).to(device)
    down, up = torch.randn(3, 8, 48, generator=gen).to(device), torch.randn(3, 56, 8, generator=gen).to(device)
    ids = torch.randint(-1, 3, (2, 30), generator=gen).to(device)
    f = _trace(lambda a, b, i, d, u: adapter_linear(a, d, u, i, base=b), x[0], base[0], ids[0], down, up)
    for k in (1, 0):
        assert torch.equal(f(x[k], base[k], ids[k], down * 2, up), adapter_linear(x[k], down * 2, up, ids[k], base=base[k]))
    at = torch.zeros(1, dtype=torch.int64, device=device)
    f = _trace(lambda a, i, o: adapter_linear(a, down, up, i, dropout_p=0.4, seed=2, offset=o), x[0], ids[0], at)
    for k in (0, 7):
        assert torch.equal(f(x[1], ids[1], at + k), adapter_linear(x[1], down, up, ids[1], dropout_p=0.4, seed=2, offset=k))
