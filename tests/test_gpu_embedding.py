"""The token embedding and its gradient by sorted tokens against 64-bit sums
(MI355X).

Bars, with u = eps / 2 of a type (half a step of rounding) and u32 = 2^-24:
the lookup rounds scale to float32, the product to float32 and that to the
weight's type, |err| <= (2 u32 + u) |ref|; a gradient row adds its n terms in
float32 in some order, (n - 1) u32 sum|g| at most, then the two roundings of
the scale and the product and that to the type.  One more u32 each covers the
products of those errors.  Below a type's smallest normal number t the numbers
lie t eps apart (float16: 2^-24), so rounding there is off by up to t eps / 2
whatever the value: |err| <= u |ref| + t eps / 2 holds for every value, and
float16, whose t is 2^-14, meets it.
"""

from __future__ import annotations

import pytest
import torch

from rosellm_amd import _native as nat
from rosellm_amd import roserlhf as R
from rosellm_amd.rosetrainer import embedding

pytestmark = pytest.mark.gpu

U32 = 2.0 ** -24
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def _bar(dtype):
    return 0.0 if dtype == torch.float32 else torch.finfo(dtype).eps / 2


def _tiny(dtype):
    f = torch.finfo(dtype)
    return f.smallest_normal * f.eps / 2


def _check_out(out, ids, w, scale, pad):
    ids = ids.reshape(-1).cpu()
    w64 = w.detach().double().cpu()
    V, H = w64.shape
    ok = (ids >= 0) & (ids < V)
    want = torch.full((ids.numel(), H), float("nan"), dtype=torch.float64)
    want[ok] = w64[ids[ok].long()] * scale
    if pad is not None:
        want[ids == pad] = 0.0
    got = out.detach().double().cpu().reshape(ids.numel(), H)
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    bar = (3 * U32 + _bar(out.dtype)) * want.abs() + _tiny(out.dtype)
    assert ((got - want).abs() <= bar).logical_or(torch.isnan(want)).all()


def _check_grad(dw, ids, g, V, scale, pad):
    H = dw.shape[1]
    ids = ids.reshape(-1).cpu().long()
    g64 = g.detach().double().cpu().reshape(ids.numel(), H)
    ok = (ids >= 0) & (ids < V)
    if pad is not None:
        ok &= ids != pad
    want = torch.zeros(V, H, dtype=torch.float64).index_add_(0, ids[ok], g64[ok]) * scale
    mass = torch.zeros(V, H, dtype=torch.float64).index_add_(0, ids[ok], g64[ok].abs()) * abs(scale)
    n = torch.bincount(ids[ok], minlength=V).double()[:, None]
    got = dw.double().cpu()
    u = _bar(dw.dtype)
    bar = (n + 3) * U32 * mass * (1 + u) + u * want.abs() + _tiny(dw.dtype)
    assert not torch.isnan(got).any()
    assert ((got - want).abs() <= bar).all(), ((got - want).abs() - bar).max()


def _ids(N, V, gen, kind):
    if kind == "even":
        return torch.randint(0, V, (N,), generator=gen)
    if kind == "one":
        return torch.full((N,), V // 2)
    # a few tokens hold most places
    return (torch.rand(N, generator=gen) ** 6 * V).long().clamp_(0, V - 1)


SIZES = [
    # N, V, H, kind
    (1, 1, 1, "even"),
    (1, 7, 3, "even"),
    (63, 5, 130, "hot"),
    (64, 5, 128, "one"),
    (65, 2, 8, "even"),
    (127, 3, 64, "one"),
    (130, 40, 1000, "hot"),
    (1000, 513, 514, "even"),
    (4096, 300, 96, "hot"),
    (4097, 50257, 33, "hot"),
    (9000, 11, 256, "even"),
    (20000, 4, 40, "one"),
    (33000, 151936, 72, "hot"),
]


@pytest.mark.parametrize("dtype", DTYPES, ids=lambda d: str(d)[6:])
@pytest.mark.parametrize("N,V,H,kind", SIZES)
def test_embedding_and_gradient(device, N, V, H, kind, dtype):
    print(f"[embedding] N={N} V={V} H={H} {kind} {dtype}", flush=True)
    gen = torch.Generator().manual_seed(N + V + H)
    ids = _ids(N, V, gen, kind)
    w = torch.randn(V, H, generator=gen).to(dtype).to(device).requires_grad_()
    g = torch.randn(N, H, generator=gen).to(dtype).to(device)
    scale = 1.0 if N % 2 else H ** 0.5
    out = embedding(ids.to(device), w, scale=scale)
    assert out.shape == (N, H) and out.dtype == dtype
    _check_out(out, ids, w, scale, None)
    out.backward(g)
    _check_grad(w.grad, ids, g, V, scale, None)
    # the same bits again
    (again,) = torch.autograd.grad(embedding(ids.to(device), w, scale=scale), w, g)
    assert torch.equal(again, w.grad)


def test_embedding_long_sort(device):
    """More positions than one block of the sort holds, ids over three passes' worth of bits."""
    gen = torch.Generator().manual_seed(5)
    V, N, H = (1 << 18) + 77, 700000, 4
    ids = torch.randint(0, V, (N,), generator=gen)
    ids[::3] = V - 1
    w = torch.zeros(V, H, device=device, requires_grad=True)
    g = torch.randn(N, H, generator=gen).to(device)
    embedding(ids.to(device), w).backward(g)
    _check_grad(w.grad, ids, g, V, 1.0, None)


@pytest.mark.parametrize("pad", [None, -1, 3])
@pytest.mark.parametrize("itype", [torch.int32, torch.int64])
def test_embedding_padding_and_bad_ids(device, pad, itype):
    gen = torch.Generator().manual_seed(9)
    V, H = 50, 24
    ids = torch.randint(0, V, (7, 31), generator=gen).to(itype)
    ids[0, :9] = torch.tensor([-1, 3, V, V + 1, -7, V - 1, 0, 3, -1])
    ids[5, 3:9] = 3
    w = torch.randn(V, H, generator=gen).to(device).requires_grad_()
    out = embedding(ids.to(device), w, scale=0.5, padding_idx=pad)
    assert out.shape == (7, 31, H)
    _check_out(out, ids, w, 0.5, pad)
    g = torch.randn(7, 31, H, generator=gen).to(device)
    g[0, 2] = float("nan")  # an id that names no row: nothing of it is read into a sum
    out.backward(g)
    _check_grad(w.grad, ids, torch.where(torch.isnan(g), 0.0, g), V, 0.5, pad)


def test_embedding_empty(device):
    w = torch.randn(6, 8, generator=torch.Generator().manual_seed(7)).to(device).requires_grad_()
    none = torch.zeros(0, 4, dtype=torch.long, device=device)
    out = embedding(none, w)
    assert out.shape == (0, 4, 8)
    out.sum().backward()
    assert torch.equal(w.grad, torch.zeros_like(w))
    all_pad = torch.full((5,), -1, device=device)
    (dw,) = torch.autograd.grad(embedding(all_pad, w, padding_idx=-1).sum(), w)
    assert torch.equal(dw, torch.zeros_like(w))
    z = torch.zeros(0, 8, device=device)
    assert torch.isnan(embedding(torch.zeros(3, dtype=torch.long, device=device), z)).all()


def test_embedding_strides(device):
    """Strided ids, a weight that is a slice or a transpose, gradients that are expanded, strided or misaligned."""
    gen = torch.Generator().manual_seed(11)
    V, H = 97, 40
    base = torch.randn(V, H + 9, generator=gen).to(torch.bfloat16).to(device)
    ids = torch.randint(0, V, (12, 10), generator=gen).to(device)
    for w in (base[:, 1:H + 1], base[:, 8:H + 8], base[:H].t(), base[::2, :H], base[:1, :H].expand(V, H)):
        w = w.detach().requires_grad_()
        i = ids.t()[::2] % w.shape[0]
        out = embedding(i, w)
        _check_out(out, i, w, 1.0, None)
        n, h = i.numel(), w.shape[1]
        for g in (torch.ones((), dtype=w.dtype, device=device).expand(n, h),
                  torch.randn(h, n, generator=gen).to(w.dtype).to(device).t(),
                  torch.randn(n, 2 * h + 1, generator=gen).to(w.dtype).to(device)[:, 1:h + 1],
                  torch.randn(1, h, generator=gen).to(w.dtype).to(device).expand(n, h)):
            (dw,) = torch.autograd.grad(embedding(i, w), w, g.reshape(*i.shape, h))
            _check_grad(dw, i, g, w.shape[0], 1.0, None)


def test_embedding_gradient_against_differences(device):
    """The map is linear in the weight: f(W + D) - f(W) = <dW, D>, here with whole numbers, so exactly."""
    gen = torch.Generator().manual_seed(13)
    ids = torch.randint(0, 30, (500,), generator=gen).to(device)
    w = torch.randint(-8, 9, (30, 16), generator=gen).float().to(device).requires_grad_()
    d = torch.randint(-8, 9, (30, 16), generator=gen).float().to(device)
    c = torch.randint(-8, 9, (500, 16), generator=gen).float().to(device)
    f = lambda x: (embedding(ids, x, scale=2.0).double() * c.double()).sum()
    (dw,) = torch.autograd.grad(f(w), w)
    assert (f(w.detach() + d) - f(w.detach())).item() == (dw.double() * d.double()).sum().item()


@pytest.mark.parametrize("N", [300, 9000])
def test_embedding_workspace_contents_do_not_matter(device, N):
    gen = torch.Generator().manual_seed(17)
    V, H = 1000, 32
    ids = torch.randint(0, V // 2, (N,), generator=gen).to(device)
    g = torch.randn(N, H, generator=gen).to(device)
    need = nat.lib().rrl_embedding_bwd_workspace_bytes(N, V, H)
    got = []
    for fill in (0, 1, 255):
        ws = torch.full((need,), fill, dtype=torch.uint8, device=device)
        dw = torch.full((V, H), float("nan"), device=device)
        nat.call("rrl_embedding_bwd", ids.data_ptr(), nat.I64, N, g.data_ptr(), nat.F32, V, H, H, 1.0, 0,
                 0, dw.data_ptr(), H, ws.data_ptr(), nat.stream_ptr(device))
        got.append(dw)
    _check_grad(got[0], ids, g, V, 1.0, None)
    assert torch.equal(got[0], got[1]) and torch.equal(got[0], got[2])


def test_embedding_captured_and_on_a_stream(device):
    """A captured lookup and gradient, replayed on new ids and gradients between eager calls on another stream."""
    gen = torch.Generator().manual_seed(19)
    V, H, N = 5000, 128, 6000
    w = torch.randn(V, H, generator=gen).to(torch.bfloat16).to(device).requires_grad_()
    ids = torch.randint(0, V, (N,), generator=gen).to(device)
    g = torch.randn(N, H, generator=gen).to(torch.bfloat16).to(device)
    side = torch.cuda.Stream(device=device)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out = embedding(ids, w, scale=2.0, padding_idx=0)
        (dw,) = torch.autograd.grad(out, w, g)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    del out, dw
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = embedding(ids, w, scale=2.0, padding_idx=0)
        (dw,) = torch.autograd.grad(out, w, g)
    for k in range(3):
        ids.copy_(torch.randint(0, V >> (3 * k), (N,), generator=gen).to(device))
        g.copy_(torch.randn(N, H, generator=gen).to(device))
        graph.replay()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            want = embedding(ids, w, scale=2.0, padding_idx=0)
            (want_dw,) = torch.autograd.grad(want, w, g)
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(dw, want_dw)
        _check_grad(dw, ids, g, V, 2.0, 0)


def test_tied_weight_step(device):
    """Both ends of a tied weight: the embedding's gradient joins the LM head's."""
    gen = torch.Generator().manual_seed(23)
    B, T, V, H = 3, 40, 1000, 64
    ids = torch.randint(0, V, (B, T + 1), generator=gen).to(device)
    w = (torch.randn(V, H, generator=gen) * 0.1).to(device).requires_grad_()
    old = torch.randn(B, T, generator=gen).mul_(0.1).sub_(7.0).to(device)
    adv = torch.randn(B, T, generator=gen).to(device)
    mask = (torch.rand(B, T, generator=gen) < 0.7).to(device)

    hidden = embedding(ids[:, :-1], w, scale=H ** 0.5)
    out = R.fused_linear_policy_loss(hidden, w, ids[:, 1:], old, adv, mask, clip_low=0.2, clip_high=0.28)
    out.loss.backward()

    w64 = w.detach().double().cpu().requires_grad_()
    i, a, m = ids.cpu(), adv.double().cpu(), mask.double().cpu()
    x = w64[i[:, :-1]] * H ** 0.5
    lp = torch.log_softmax(x @ w64.t(), -1).gather(-1, i[:, 1:, None]).squeeze(-1)
    ratio = torch.exp(lp - old.double().cpu())
    loss = -(torch.minimum(ratio * a, ratio.clamp(0.8, 1.28) * a) * m).sum() / m.sum()
    loss.backward()
    scale = w64.grad.abs().max().item()
    # float32 products of H and sums of V terms: their worst-case growth, 64 + 1000 roundings, of the largest entry
    assert abs(out.loss.item() - loss.item()) <= 1064 * U32 * max(1.0, abs(loss.item()))
    assert (w.grad.double().cpu() - w64.grad).abs().max().item() <= 1064 * U32 * scale
