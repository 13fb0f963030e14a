"""Dropout from a counter-based generator against the mask's definition (MI355X).

Bars, with u = eps / 2 of the type (half a step of rounding) and u32 = 2^-24: the scale
is rounded to float32, the product (or its sum with the residual) to float32 and that to
the type: |err| <= u32 |x s| + u32 |y| + u |y|, and one u32 |x s| + u32 |y| more for the
products of those errors; plus half a step below the type's smallest normal number.
"""

from __future__ import annotations

import pytest
import torch

from rosellm_amd.rosetrainer import dropout, embedding

from _philox import keep

pytestmark = pytest.mark.gpu

U32 = 2.0 ** -24
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def _check(y, x, res, mask, scale):
    f = torch.finfo(y.dtype)
    x64 = x.detach().double().cpu().reshape(mask.shape)
    add = torch.where(mask, x64 * scale, 0.0)
    want = add if res is None else add + res.detach().double().cpu().reshape(mask.shape)
    got = y.detach().double().cpu().reshape(mask.shape)
    u = 0.0 if y.dtype == torch.float32 else f.eps / 2
    bar = 2 * U32 * add.abs() + (2 * U32 + u) * want.abs() + f.smallest_normal * f.eps / 2
    assert ((got - want).abs() <= bar).all(), ((got - want).abs() - bar).max()
    if res is None:  # dropped entries are zeros, not small numbers
        assert torch.equal(got == 0, ~mask | (x64 == 0))


@pytest.mark.parametrize("dtype", DTYPES, ids=lambda d: str(d)[6:])
@pytest.mark.parametrize("shape", [(1,), (7,), (8,), (9,), (1, 1), (3, 8), (5, 770), (2, 3, 64), (130, 33), (1000, 1),
                                   (63, 1024), (4097, 40)], ids=str)
@pytest.mark.parametrize("p", [0.0, 0.1, 0.5])
def test_mask_value_and_gradient(device, shape, dtype, p):
    print(f"[dropout] {shape} {dtype} {p}", flush=True)
    gen = torch.Generator().manual_seed(sum(shape))
    x = torch.randn(shape, generator=gen).to(dtype).to(device).requires_grad_()
    res = torch.randn(shape, generator=gen).to(dtype).to(device).requires_grad_()
    g = torch.randn(shape, generator=gen).to(dtype).to(device)
    cols = shape[-1]
    rows = x.numel() // cols
    for seed, offset, r in ((3, 0, None), (2 ** 63 + 5, 2 ** 33 + 1, res), (-1, -1, res)):
        mask, scale = keep(rows, cols, p, seed, offset)
        y = dropout(x, p, seed=seed, offset=offset, residual=r)
        assert y.shape == x.shape and y.dtype == dtype
        _check(y, x, r, mask, scale)
        grads = torch.autograd.grad(y, [x] if r is None else [x, r], g)
        _check(grads[0], g, None, mask, scale)
        if r is not None:
            assert torch.equal(grads[1], g)


def test_probabilities(device):
    """All kept, none kept, thresholds between two steps, and the share that is kept."""
    x = torch.ones(1 << 20, device=device)
    assert torch.equal(dropout(x, 0.0, seed=1), x)
    assert not dropout(x, 1.0, seed=1).any()
    assert not dropout(x, 1.0 - 2.0 ** -18, seed=1).any()  # rounds to 1
    for p in (2.0 ** -18, 2.0 ** -16, 0.3, 0.999):
        y = dropout(x, p, seed=9, offset=4).cpu()
        mask, scale = keep(1, 1 << 20, p, 9, 4)
        assert torch.equal(y != 0, mask[0])
        assert (y[mask[0]] == torch.tensor(scale, dtype=torch.float32)).all()
    # of 2^20 entries the share kept is within five deviations of sqrt(0.25 / 2^20) / ...
    y = dropout(x, 0.5, seed=11)
    assert abs(float((y != 0).double().mean()) - 0.5) < 5 * (0.25 / 2 ** 20) ** 0.5


def test_dropped_entries_are_zero_whatever_they_were(device):
    x = torch.full((4, 64), float("nan"), device=device)
    x[1] = float("inf")
    mask, _ = keep(4, 64, 0.5, 3, 0)
    y = dropout(x, 0.5, seed=3).cpu()
    assert torch.equal(y == 0, ~mask)
    r = torch.ones_like(x)
    assert torch.equal(dropout(x, 0.5, seed=3, residual=r).cpu() == 1, ~mask)


def test_strides_and_offsets(device):
    """Transposed, sliced, expanded and odd-addressed operands give what their copies give."""
    gen = torch.Generator().manual_seed(0)
    big = torch.randn(40, 70, generator=gen).to(torch.bfloat16).to(device)
    views = [big.t(), big[:, 3:61], big[1::2, 1:], big[:, :1].expand(40, 70), big[:1].expand(40, 70), big[:, ::2],
             big.reshape(4, 10, 70).transpose(0, 1), big.flatten()[1:1 + 33 * 17].view(33, 17)]
    for v in views:
        for r in (None, v.flip(0)):
            a = dropout(v, 0.25, seed=5, residual=r)
            b = dropout(v.contiguous(), 0.25, seed=5, residual=None if r is None else r.contiguous())
            assert torch.equal(a, b) and a.is_contiguous()
    # a gradient that is one number, expanded
    x = torch.ones(6, 33, device=device, requires_grad=True)
    dropout(x, 0.5, seed=2).sum().backward()
    mask, scale = keep(6, 33, 0.5, 2, 0)
    assert torch.equal(x.grad.cpu(), mask.float() * scale)


def test_empty(device):
    for shape in ((0,), (0, 5), (3, 0)):
        x = torch.zeros(shape, device=device, requires_grad=True)
        y = dropout(x, 0.5, seed=1)
        assert y.shape == shape
        y.sum().backward()
        assert x.grad.shape == shape
    assert float(dropout(torch.tensor(2.0, device=device), 0.0)) == 2.0


def test_offset_on_the_device(device):
    """The offset read by the kernel; changed before the backward, it raises there."""
    x = torch.randn(64, 96, device=device, requires_grad=True)
    at = torch.tensor([7], device=device)
    y = dropout(x, 0.5, seed=4, offset=at)
    assert torch.equal(y, dropout(x, 0.5, seed=4, offset=7))
    (g,) = torch.autograd.grad(y, x, torch.ones_like(y))
    assert torch.equal(g != 0, y != 0)
    y = dropout(x, 0.5, seed=4, offset=at)
    at.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(y, x, torch.ones_like(y))


def test_captured(device):
    """A captured call draws another mask at each replay through its offset; eager work between the replays."""
    x = torch.randn(256, 520, device=device)
    at = torch.zeros(1, dtype=torch.int64, device=device)
    dropout(x, 0.1, seed=6, offset=at)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = dropout(x, 0.1, seed=6, offset=at, residual=x)
        at.add_(1)
    seen = []
    for k in range(4):
        x.normal_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, dropout(x, 0.1, seed=6, offset=k, residual=x))
        seen.append(y != x)
    assert not torch.equal(seen[0], seen[1])


def test_streams_and_seeds(device):
    x = torch.randn(300, 1000, device=device)
    want = dropout(x, 0.2, seed=1)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = dropout(x, 0.2, seed=1)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    # seeds drawn from a host generator
    a = dropout(x, 0.2, generator=torch.Generator().manual_seed(8))
    b = dropout(x, 0.2, generator=torch.Generator().manual_seed(8))
    c = dropout(x, 0.2, generator=torch.Generator().manual_seed(9))
    assert torch.equal(a, b) and not torch.equal(a, c)


def test_differences(device):
    """The loss is linear in x: its change along v is the gradient times v.

    loss = sum(g y); every y is off by 3 u32 |y|, so the two losses by 3 u32 sum |g y| each."""
    gen = torch.Generator().manual_seed(4)
    x, v, g = (torch.randn(50, 77, generator=gen).to(device) for _ in range(3))
    xr = x.clone().requires_grad_()
    (dx,) = torch.autograd.grad(dropout(xr, 0.3, seed=3), xr, g)
    up, down = dropout(x + v, 0.3, seed=3), dropout(x - v, 0.3, seed=3)
    change = (g.double() * (up.double() - down.double())).sum() / 2
    step = ((x + v).double() - (x - v).double()) / 2  # what was moved, with its rounding
    want = (dx.double() * step).sum()
    bar = 3 * U32 * (g.double().abs() * (up.double().abs() + down.double().abs()) / 2).sum() + 3 * U32 * (
        dx.double() * step).abs().sum()
    assert (change - want).abs() <= bar


def test_after_the_embedding(device):
    """Rows of the embedding, dropped out; equal to dropping the gradient's rows."""
    gen = torch.Generator().manual_seed(2)
    ids = torch.randint(0, 50, (12, 30), generator=gen).to(device)
    w = torch.randn(50, 72, generator=gen).to(device).requires_grad_()
    g = torch.randn(12, 30, 72, generator=gen).to(device)
    out = dropout(embedding(ids, w, scale=2.0), 0.1, seed=7)
    (dw,) = torch.autograd.grad(out, w, g)
    dropped = dropout(g, 0.1, seed=7)
    (want,) = torch.autograd.grad(embedding(ids, w, scale=2.0), w, dropped)
    assert torch.equal(dw, want)


def test_without_a_graph(device):
    """A call that nothing differentiates gives the recorded call's bits; forward mode is refused."""
    x, r = torch.randn(9, 50, device=device), torch.randn(9, 50, device=device)
    y = dropout(x, 0.3, seed=1, residual=r)
    assert y.grad_fn is None
    for a, b in ((x.clone().requires_grad_(), r), (x, r.clone().requires_grad_())):
        z = dropout(a, 0.3, seed=1, residual=b)
        assert z.grad_fn is not None and torch.equal(y, z)
        with torch.no_grad():
            z = dropout(a, 0.3, seed=1, residual=b)
        assert z.grad_fn is None and torch.equal(y, z)
    import torch.autograd.forward_ad as fwd
    with fwd.dual_level(), pytest.raises((RuntimeError, NotImplementedError)):
        dropout(fwd.make_dual(x, torch.ones_like(x)), 0.3, seed=1)
