"""The largest sizes that adapters are taken of (MI355X)."""

from __future__ import annotations

import pytest
import torch

from rosellm_amd.rosetrainer import adapter_linear

from test_gpu_adapters import _close, _reference

pytestmark = [pytest.mark.gpu, pytest.mark.slow]


@pytest.fixture(autouse=True)
def _release():
    yield
    torch.cuda.empty_cache()


def test_gradients_of_over_2_to_the_30_weights(device):
    """Four threads to each of them are more than a grid can have."""
    N, A, H, O, r = 40, 64, 1024, 131072, 128
    assert 4 * A * r * (H + O) > 1 << 32
    gen = torch.Generator(device="cuda").manual_seed(1)
    rand = lambda *s: torch.randn(*s, generator=gen, device=device, dtype=torch.bfloat16)
    x, g = rand(N, H), rand(N, O)
    down, up = rand(A, r, H).mul_(H ** -0.5).requires_grad_(), rand(A, O, r).requires_grad_()
    pick = torch.tensor([0, 31, 63], device=device)
    at = torch.randint(0, 3, (N,), generator=gen, device=device)
    y = adapter_linear(x, down, up, pick[at])
    dd, du = torch.autograd.grad(y, (down, up), g)
    want = _reference(x, None, down.detach()[pick], up.detach()[pick], at, g, None)
    for got, (w, e), what in ((y, want[0], "y"), (dd[pick], want[2], "ddown"), (du[pick], want[3], "dup")):
        _close(got, w.cpu(), e.cpu(), what)
    others = torch.ones(A, dtype=torch.bool, device=device)
    others[pick] = False
    assert not dd[others].any()
    for a in others.nonzero().flatten().tolist():
        assert not du[a].any(), a


@pytest.mark.parametrize("N,r", [(1 << 30, 3), ((1 << 28) + 77, 70)])
def test_most_rows(device, N, r):
    """Rows of one entry: t alone takes 69 GB for 2^30 rows of rank 16, and 137 for a quarter of them of rank 128."""
    x = torch.zeros(N, 1, dtype=torch.bfloat16, device=device)
    some = torch.cat([torch.arange(0, 3000), torch.arange(N // 2, N // 2 + 3000), torch.arange(N - 3000, N)]).to(device)
    x[some] = (torch.arange(9000, device=device) % 251 - 125).bfloat16()[:, None]
    down, up = torch.zeros(1, r, 1, device=device).bfloat16(), torch.zeros(1, 1, r, device=device).bfloat16()
    down[0, r - 1], up[0, 0, r - 1] = 0.5, 4.0
    y = adapter_linear(x, down, up)
    assert y.shape == (N, 1)
    assert torch.equal(y, x * 2)
