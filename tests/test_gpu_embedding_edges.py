"""The embedding's largest rows (MI355X): the bars are test_gpu_embedding's."""

from __future__ import annotations

import pytest
import torch

from rosellm_amd.rosetrainer import embedding

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=lambda d: str(d)[6:])
def test_embedding_widest_rows(device, dtype):
    """Rows of 2^22 - 1 elements, whose odd length allows single-element accesses only."""
    print(f"[embedding] widest {dtype}", flush=True)
    V, H = 3, (1 << 22) - 1
    gen = torch.Generator(device=device).manual_seed(29)
    w = torch.randn(V, H, generator=gen, device=device).to(dtype).requires_grad_()
    ids = torch.tensor([2, 0, 2], device=device)
    # whole numbers, so that sums are exact
    g = torch.randint(-8, 9, (3, H), generator=gen, device=device).to(dtype)
    out = embedding(ids, w, scale=2.0)
    assert torch.equal(out, w.detach()[ids] * 2)
    (dw,) = torch.autograd.grad(out, w, g)
    assert torch.equal(dw, torch.stack([g[1] * 2, torch.zeros_like(g[0]), (g[0] + g[2]) * 2]))


def test_embedding_long_runs_of_wide_rows(device):
    """Runs of more than 64 positions over rows of many columns' shares, at every access width."""
    gen = torch.Generator(device=device).manual_seed(31)
    V, N = 3, 700
    ids = (torch.rand(N, generator=gen, device=device) * 1.4).long()
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        for H in (1024, 1028, 1030, 1031):
            g = torch.randint(-2, 3, (N, H), generator=gen, device=device).to(dtype)
            w = torch.zeros(V, H, dtype=dtype, device=device, requires_grad=True)
            (dw,) = torch.autograd.grad(embedding(ids, w), w, g)
            want = torch.stack([g[ids == v].double().sum(0) for v in range(V)])
            # whole numbers up to 1400: exact sums, rounded once
            assert torch.equal(dw, want.to(dtype)), (dtype, H)
