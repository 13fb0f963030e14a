"""What stands between an adapter's two products is held to all of float32's 24 bits (MI355X).

The operands are chosen so that every sum of them is a number of at most 24 bits and the
result is the last of these bits alone: results are equal, and a t (or s) of fewer bits
gives none of them right."""

from __future__ import annotations

import pytest
import torch

from rosellm_amd.rosetrainer import adapter_linear

pytestmark = pytest.mark.gpu

# three numbers of the type that fill 24 bits side by side, and what the last one is divided by to stay in its range
PARTS = {
    torch.bfloat16: (1 + 2.0 ** -7, 2.0 ** -8 * (1 + 2.0 ** -7), 2.0 ** -17 * (1 + 2.0 ** -6), 1.0),
    torch.float16: (1 + 2.0 ** -10, 2.0 ** -11 * (1 + 2.0 ** -10), 2.0 ** -22 * 1.5, 2.0 ** -10),
    torch.float32: (1 + 2.0 ** -7, 2.0 ** -8 * (1 + 2.0 ** -7), 2.0 ** -17 * (1 + 2.0 ** -6), 1.0),
}
RANKS = [2, 16, 17, 40, 64, 100, 128]
# one launch, two launches of few rows, and many rows
ROWS = [(3, 40), (3, 16400), (1500, 40), (1500, 256)]


def _ids(dtype):
    return str(dtype)[6:]


@pytest.mark.parametrize("dtype", list(PARTS), ids=_ids)
@pytest.mark.parametrize("r", RANKS)
@pytest.mark.parametrize("N,O", ROWS)
def test_the_product(device, N, O, r, dtype):
    """t of two ranks, which differ in the last part alone, subtracted by up."""
    H = 256 if O == 256 else 72
    h, m, l, low = PARTS[dtype]
    at = [3, 33, H - 1]
    x = torch.zeros(N, H)
    x[:, at] = torch.tensor([1.0, 1.0, low])
    down = torch.zeros(2, r, H)
    down[:, r - 2, at] = torch.tensor([h, m, l / low])
    down[:, r - 1, at] = torch.tensor([h, m, 0.0])
    up = torch.zeros(2, O, r)
    c = 1.0 + (2.0 ** -9 if dtype == torch.float16 else 0.0)  # with bits past bfloat16's eight
    up[:, :, r - 2], up[:, :, r - 1] = c, -c
    ids = torch.arange(N) % 2
    scales = torch.tensor([2.0 ** 10, 2.0 ** 11])
    x, down, up, ids, scales = (v.to(device) for v in (x.to(dtype), down.to(dtype), up.to(dtype), ids, scales))
    y = adapter_linear(x, down, up, ids, scales=scales)
    want = (scales[ids] * c * l).to(dtype)[:, None].expand(N, O)
    assert (want.double() == scales[ids].double()[:, None] * c * l).all()
    assert torch.equal(y, want)


@pytest.mark.parametrize("dtype", list(PARTS), ids=_ids)
@pytest.mark.parametrize("r", RANKS)
@pytest.mark.parametrize("N,H", ROWS)
def test_the_gradient_of_x(device, N, H, r, dtype):
    """The same of s = up^T g."""
    O = 256 if H == 256 else 72
    h, m, l, low = PARTS[dtype]
    at = [3, 33, O - 1]
    g = torch.zeros(N, O)
    g[:, at] = torch.tensor([1.0, 1.0, low])
    up = torch.zeros(1, O, r)
    up[0, at, r - 2] = torch.tensor([h, m, l / low])
    up[0, at, r - 1] = torch.tensor([h, m, 0.0])
    down = torch.zeros(1, r, H)
    c = 1.0 + (2.0 ** -9 if dtype == torch.float16 else 0.0)
    down[:, r - 2], down[:, r - 1] = c, -c
    x = torch.ones(N, H).to(dtype).to(device).requires_grad_()
    y = adapter_linear(x, down.to(dtype).to(device), up.to(dtype).to(device), scales=torch.tensor([2.0 ** 10], device=device))
    (dx,) = torch.autograd.grad(y, x, g.to(dtype).to(device))
    assert torch.equal(dx, torch.full((N, H), 2.0 ** 10 * c * l, dtype=dtype, device=device))


@pytest.mark.parametrize("dtype", list(PARTS), ids=_ids)
@pytest.mark.parametrize("r", RANKS)
@pytest.mark.parametrize("N", [2, 70, 1500])
def test_the_factors_gradients(device, N, r, dtype):
    """Sums over two tokens of opposite signs, whose t and s differ in the last part alone."""
    h, m, l, low = PARTS[dtype]
    H = O = 72
    at = [3, 33, H - 1]
    c = 1.0 + (2.0 ** -9 if dtype == torch.float16 else 0.0)
    i, j = 0, min(N - 1, 20)  # of one run of tokens
    scales = torch.tensor([2.0 ** 10], device=device)
    # s: h + m + l of token i, h + m of token j, beside x of c and -c
    g, up, x = torch.zeros(N, O), torch.zeros(1, O, r), torch.zeros(N, H)
    g[i, at], g[j, at] = torch.tensor([1.0, 1.0, low]), torch.tensor([1.0, 1.0, 0.0])
    up[0, at, r - 1] = torch.tensor([h, m, l / low])
    x[i], x[j] = c, -c
    leaves = [v.to(dtype).to(device) for v in (x, torch.zeros(1, r, H), up)]
    leaves[1].requires_grad_()
    (dd,) = torch.autograd.grad(adapter_linear(*leaves, scales=scales), leaves[1], g.to(dtype).to(device))
    want = torch.zeros(1, r, H, dtype=dtype, device=device)
    want[:, r - 1] = 2.0 ** 10 * c * l
    assert torch.equal(dd, want)
    # t: the same of x, beside g of c and -c
    x, down, g = torch.zeros(N, H), torch.zeros(1, r, H), torch.zeros(N, O)
    x[i, at], x[j, at] = torch.tensor([1.0, 1.0, low]), torch.tensor([1.0, 1.0, 0.0])
    down[0, r - 1, at] = torch.tensor([h, m, l / low])
    g[i], g[j] = c, -c
    leaves = [v.to(dtype).to(device) for v in (x, down, torch.zeros(1, O, r))]
    leaves[2].requires_grad_()
    (du,) = torch.autograd.grad(adapter_linear(*leaves, scales=scales), leaves[2], g.to(dtype).to(device))
    want = torch.zeros(1, O, r, dtype=dtype, device=device)
    want[:, :, r - 1] = 2.0 ** 10 * c * l
    assert torch.equal(du, want)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=_ids)
@pytest.mark.parametrize("r", [3, 20])
@pytest.mark.parametrize("N", [2, 1500])
def test_a_product_next_to_float32s_largest(device, N, r, dtype):
    """t above the largest bfloat16, to which it would round up to infinity."""
    big = torch.finfo(torch.bfloat16).max
    x = torch.zeros(N, 8)
    x[:, :2] = torch.tensor([big, 2.0 ** 119 * 1.5])
    down, up = torch.zeros(1, r, 8), torch.zeros(1, 16, r)
    down[0, 0, :2] = 1.0
    up[0, :, 0] = 2.0 ** -100
    y = adapter_linear(x.to(dtype).to(device), down.to(dtype).to(device), up.to(dtype).to(device))
    want = torch.tensor((big + 2.0 ** 119 * 1.5) * 2.0 ** -100, dtype=torch.float64).to(dtype)
    assert float(want) > 0 and torch.equal(y.cpu(), want.expand(N, 16))
