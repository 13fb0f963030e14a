"""Operands of more than 2^32 elements, or whose parts lie that far apart: the same
results as on small operands (MI355X)."""

from __future__ import annotations

import pytest
import torch

from rosellm_amd import roseinfer as RI
from rosellm_amd.rosetrainer import embedding

pytestmark = pytest.mark.gpu

FAR = 1 << 32


@pytest.fixture(autouse=True)
def _room():
    yield
    torch.cuda.empty_cache()


def test_verify_far_rows(device):
    g = torch.Generator().manual_seed(37)
    B, K, V = 2, 2, 3001
    x = (torch.randn(B, K + 1, V, generator=g) * 2).to(torch.bfloat16).to(device)
    y = (x[:, :K].float() + 0.5).to(torch.bfloat16)
    d = y.float().argmax(-1)
    u = torch.rand(B, K + 1, generator=g).to(device)
    base = torch.empty(FAR + 3 * (FAR // 4) + 8192, dtype=torch.bfloat16, device=device)
    far_x = base.as_strided((B, K + 1, V), (FAR + 11, FAR // 4, 1), 5)
    far_y = base.as_strided((B, K, V), (FAR + 11, FAR // 4, 1), 4001)
    far_x.copy_(x)
    far_y.copy_(y)
    for q, far_q in ((y, far_y), (None, None)):
        want = RI.verify_draft_tokens(x, d, q, u)
        got = RI.verify_draft_tokens(far_x, d, far_q, u)
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_quantize_far_rows(device):
    R, H = (1 << 20) + 1, 4100
    x = torch.empty(R, H, dtype=torch.float16, device=device).uniform_(-4, 4, generator=torch.Generator(device=device).manual_seed(41))
    assert x.numel() > FAR
    q = RI.quantize_mxfp4(x)
    back = RI.dequantize_mxfp4(q, torch.float16)
    for lo in (0, R // 2, R - 300):
        part = RI.quantize_mxfp4(x[lo:lo + 300])
        assert torch.equal(q.codes[lo:lo + 300], part.codes) and torch.equal(q.scales[lo:lo + 300], part.scales)
        assert torch.equal(back[lo:lo + 300], RI.dequantize_mxfp4(part, torch.float16))


@pytest.mark.parametrize("N", [220000, 220001])  # whole vectors, and rows at odd addresses
def test_linear_far_rows(device, N):
    M, H = 20000, 128
    g = torch.Generator(device=device).manual_seed(43)
    x = torch.randn(M, H, generator=g, device=device).to(torch.bfloat16)
    q = RI.quantize_mxfp4(torch.randn(N, H, generator=g, device=device))
    out = RI.mxfp4_linear(x, q)
    assert out.numel() > FAR
    for lo in (0, M // 2, M - 70):
        # one instruction's depth: the sums' order does not depend on the rows beside
        assert torch.equal(out[lo:lo + 70], RI.mxfp4_linear(x[lo:lo + 70], q))


def test_embedding_far_rows(device):
    V, H, N = 61, 2048, (1 << 21) + 3
    g = torch.Generator(device=device).manual_seed(47)
    w = torch.randn(V, H, generator=g, device=device).to(torch.bfloat16).requires_grad_()
    ids = torch.randint(0, V, (N,), generator=g, device=device)
    out = embedding(ids, w, scale=2.0)
    assert out.numel() > FAR
    for lo in (0, N // 2, N - 1000):
        assert torch.equal(out[lo:lo + 1000], w.detach()[ids[lo:lo + 1000]] * 2)
    grad = torch.empty(N, H, dtype=torch.bfloat16, device=device).random_(0, 4, generator=g)
    (dw,) = torch.autograd.grad(out, w, grad)
    want = torch.zeros(V, H, device=device)
    for lo in range(0, N, 1 << 17):  # whole numbers up to 2^18: exact in float32
        want.index_add_(0, ids[lo:lo + (1 << 17)], grad[lo:lo + (1 << 17)].float())
    assert torch.equal(dw, (want * 2).to(torch.bfloat16))
