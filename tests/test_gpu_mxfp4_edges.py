"""The 4-bit product's operands at addresses of their own (MI355X)."""

from __future__ import annotations

import pytest
import torch

from rosellm_amd import roseinfer as RI

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("offset", [1, 2, 3, 4])
@pytest.mark.parametrize("M,N,H", [(3, 200, 96), (40, 264, 700), (5, 130, 1500)])
def test_scales_at_any_address(device, M, N, H, offset):
    """Scales held as a view at any byte give the bits that they give by themselves."""
    print(f"[mxfp4] M={M} N={N} H={H} scales at {offset}", flush=True)
    g = torch.Generator().manual_seed(M + N + H)
    q = RI.quantize_mxfp4((torch.randn(N, H, generator=g) * torch.exp(torch.randn(N, 1, generator=g))).to(device))
    x = torch.randn(M, H, generator=g).to(device)
    room = torch.full((q.scales.numel() + 16,), 255, dtype=torch.uint8, device=device)
    view = room[offset:offset + q.scales.numel()].view(q.scales.shape)
    view.copy_(q.scales)
    assert view.data_ptr() % 4 == offset % 4
    moved = RI.MxFp4(q.codes, view, q.cols)
    assert torch.equal(RI.mxfp4_linear(x, moved), RI.mxfp4_linear(x, q))
    assert torch.equal(RI.dequantize_mxfp4(moved), RI.dequantize_mxfp4(q))
