"""Low-rank adapters of many requests and their gradients against 64-bit products (MI355X).

Bars, with u = eps / 2 of the type (half a step of rounding) and u32 = 2^-24, products of
two numbers of a type exact for 16-bit types, and an addition in the matrix unit off by
at most a whole step (2 u32), the operands' products of float32 by another:
  t = down x (H terms): e_t = 2 (H + 8) u32 |down| |x|, and 2^-16 |t| more where the second
    product takes it in two parts (16-bit types: 2^-17, and of float16 2^-18 that is left out)
  y: |scale| (|up| e_t + 2 (3 r + 8) u32 |up| |t|) + 3 u32 |y| + u |y|
The gradients' products have the same form, with n rows in place of H or r.  Half a step
below the type's smallest normal number comes on top.
"""

from __future__ import annotations

import pytest
import torch
import torch.nn.functional as F

from rosellm_amd.rosetrainer import adapter_linear, dropout
from rosellm_amd.roseinfer import sample_tokens
from rosellm_amd import roserlhf as R

from _philox import keep

pytestmark = pytest.mark.gpu

U32 = 2.0 ** -24
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def _make(N, A, H, O, r, dtype, gen, runs=1, none=0.15):
    x = torch.randn(N, H, generator=gen).to(dtype)
    base = torch.randn(N, O, generator=gen).to(dtype)
    down = (torch.randn(A, r, H, generator=gen) * H ** -0.5).to(dtype)
    up = torch.randn(A, O, r, generator=gen).to(dtype)
    n = -(-N // runs)
    ids = torch.randint(0, A, (n,), generator=gen)
    ids = torch.where(torch.rand(n, generator=gen) < none, -1, ids).repeat_interleave(runs)[:N]
    g = torch.randn(N, O, generator=gen).to(dtype)
    return x, base, down, up, ids, g


def _close(got, want, err, what):
    f = torch.finfo(got.dtype)
    u = 0.0 if got.dtype == torch.float32 else f.eps / 2
    got = got.detach().double().cpu()
    bar = err + (3 * U32 + u) * want.abs() * (1 + 2 * u) + u * err + f.smallest_normal * f.eps / 2
    assert not torch.isnan(got).any(), what
    assert ((got - want).abs() <= bar).all(), (what, ((got - want).abs() - bar).max(), want.abs().max())


def _reference(x, base, down, up, ids, g, scales, mask=None, factor=1.0):
    """Each output in 64 bits with what it may be off by, before its rounding."""
    f64 = [v.double() for v in (x, down, up)]
    xd, dd, ud = f64
    if mask is not None:
        xd = torch.where(mask, xd * factor, 0.0)
    N, A = x.shape[0], down.shape[0]
    H, r, O = dd.shape[2], dd.shape[1], ud.shape[1]
    low = 0.0 if x.dtype == torch.float32 else 2.0 ** -16
    new = lambda c: torch.zeros(N, c, dtype=torch.float64, device=x.device)
    y = new(O) if base is None else base.double().clone()
    ey, dx, edx = new(O), new(H), new(H)
    ddown, eddown, dup, edup = (torch.zeros_like(v) for v in (dd, dd, ud, ud))
    for a in range(A):
        n = (ids == a).nonzero().flatten()
        if n.numel() == 0:
            continue
        s = 1.0 if scales is None else float(scales[a])
        xa, k = xd[n], n.numel()
        t, ta = xa @ dd[a].T, xa.abs() @ dd[a].abs().T
        et = 2 * (H + 8) * U32 * ta + low * t.abs()
        y[n] += s * (t @ ud[a].T)
        ey[n] = abs(s) * (et @ ud[a].abs().T + 2 * (3 * r + 8) * U32 * (t.abs() @ ud[a].abs().T))
        if g is None:
            continue
        ga = g[n].double()
        b, ba = ga @ ud[a], ga.abs() @ ud[a].abs()
        eb = 2 * (O + 8) * U32 * ba + low * b.abs()
        m = torch.ones_like(xa) if mask is None else mask[n].double() * factor
        dx[n] = s * (b @ dd[a]) * m
        edx[n] = abs(s) * (eb @ dd[a].abs() + 2 * (3 * r + 8) * U32 * (b.abs() @ dd[a].abs())) * m
        ddown[a] = s * (b.T @ xa)
        eddown[a] = abs(s) * (eb.T @ xa.abs() + 2 * (3 * k + 300) * U32 * (b.abs().T @ xa.abs()))
        dup[a] = s * (ga.T @ t)
        edup[a] = abs(s) * (ga.abs().T @ et + 2 * (3 * k + 300) * U32 * (ga.abs().T @ t.abs()))
    return (y, ey), (dx, edx), (ddown, eddown), (dup, edup)


def _run(device, x, base, down, up, ids, g, scales, **kw):
    leaves = [v.to(device).requires_grad_() for v in (x, down, up)]
    b = None if base is None else base.to(device).requires_grad_()
    y = adapter_linear(*leaves, ids.to(device), base=b, scales=None if scales is None else scales.to(device), **kw)
    if g is None:
        return (y,)
    grads = torch.autograd.grad(y, leaves + ([] if b is None else [b]), g.to(device))
    if b is not None:
        assert torch.equal(grads[3].cpu(), g)
    return (y, *grads[:3])


CASES = [
    # N, A, H, O, r, runs
    (1, 1, 1, 1, 1, 1),
    (1, 3, 64, 48, 4, 1),
    (2, 1, 7, 9, 3, 1),
    (15, 4, 40, 33, 8, 1),
    (16, 2, 32, 32, 16, 1),
    (17, 2, 33, 130, 17, 1),
    (64, 16, 128, 96, 16, 1),
    (65, 5, 1000, 70, 5, 1),
    (100, 1, 96, 257, 32, 100),
    (255, 40, 72, 40, 9, 1),
    (257, 3, 136, 64, 64, 50),
    (300, 2, 50, 1030, 33, 7),
    (1023, 7, 48, 24, 12, 1),
    (1025, 2, 520, 16, 16, 300),
    (2500, 3, 65, 67, 24, 1),
    (3000, 1, 64, 640, 128, 3000),
    (130, 3, 257, 90, 100, 1),
    (700, 300, 16, 24, 2, 1),
]


@pytest.mark.parametrize("dtype", DTYPES, ids=lambda d: str(d)[6:])
@pytest.mark.parametrize("N,A,H,O,r,runs", CASES)
def test_product_and_gradients(device, N, A, H, O, r, runs, dtype):
    print(f"[adapters] N={N} A={A} H={H} O={O} r={r} runs={runs} {dtype}", flush=True)
    gen = torch.Generator().manual_seed(N + H + r)
    x, base, down, up, ids, g = _make(N, A, H, O, r, dtype, gen, runs)
    scales = torch.rand(A, generator=gen) * 2 + 0.1
    for b, s, p in ((base, scales, 0.0), (None, None, 0.0), (base, scales, 0.2)):
        kw = dict(dropout_p=p, seed=5, offset=3) if p else {}
        mask, factor = keep(N, H, p, 5, 3) if p else (None, 1.0)
        out = _run(device, x, b, down, up, ids, g, s, **kw)
        want = _reference(x, b, down, up, ids, g, s, mask, factor)
        for got, (w, e), what in zip(out, want, ("y", "dx", "ddown", "dup")):
            assert got.dtype == dtype and got.shape == w.shape
            _close(got, w, e, what)
        # rows without an adapter are the base's, bit for bit, and pass nothing
        none = ids < 0
        assert torch.equal(out[0][none.to(device)].cpu(), torch.zeros_like(base)[none] if b is None else base[none])
        assert not out[1][none.to(device)].any()
        # the same bits again
        again = _run(device, x, b, down, up, ids, g, s, **kw)
        for p1, p2 in zip(out, again):
            assert torch.equal(p1, p2)


def test_only_what_is_asked_for(device):
    """Each gradient alone is the same as with the others, and frozen operands take none."""
    gen = torch.Generator().manual_seed(3)
    x, base, down, up, ids, g = _make(333, 3, 80, 56, 10, torch.bfloat16, gen, 20)
    want = _run(device, x, base, down, up, ids, g, None, dropout_p=0.1, seed=2)
    gd, idd = g.to(device), ids.to(device)
    for i in range(3):
        leaves = [v.to(device) for v in (x, down, up)]
        leaves[i].requires_grad_()
        y = adapter_linear(*leaves, idd, base=base.to(device), dropout_p=0.1, seed=2)
        assert torch.equal(y, want[0])
        assert torch.equal(torch.autograd.grad(y, leaves[i], gd)[0], want[1 + i])
    with torch.no_grad():
        assert torch.equal(adapter_linear(x.to(device), down.to(device), up.to(device), idd, base=base.to(device),
                                          dropout_p=0.1, seed=2), want[0])
    y = adapter_linear(x.to(device), down.to(device), up.to(device), idd)
    assert not y.requires_grad


def test_ids(device):
    """int32, no ids, all negative, ids that there are none of, and adapters without rows."""
    gen = torch.Generator().manual_seed(4)
    x, base, down, up, ids, g = _make(200, 4, 64, 48, 8, torch.float32, gen)
    a = _run(device, x, base, down, up, ids, g, None)
    b = _run(device, x, base, down, up, ids.int(), g, None)
    for p, q in zip(a, b):
        assert torch.equal(p, q)
    one = adapter_linear(x.to(device), down[:1].to(device), up[:1].to(device), base=base.to(device))
    zero = adapter_linear(x.to(device), down.to(device), up.to(device), torch.zeros(200, dtype=torch.long, device=device),
                          base=base.to(device))
    assert torch.equal(one, zero)
    y, dx, dd, du = _run(device, x, base, down, up, torch.full((200,), -5), g, None)
    assert torch.equal(y.cpu(), base) and not dx.any() and not dd.any() and not du.any()
    bad = ids.clone()
    bad[::7] = 4
    bad[3] = 2 ** 40
    there = (bad < 4) | (bad < 0)
    out = _run(device, x, base, down, up, bad, g, None)
    assert torch.isnan(out[0].cpu()[~there]).all() and not torch.isnan(out[0].cpu()[there]).any()
    assert not out[1].cpu()[~there].any()
    want = _reference(x, base, down, up, torch.where(there, bad, -1), g, None)
    for got, (w, e), what in list(zip(out, want, ("y", "dx", "ddown", "dup")))[1:]:
        _close(got, w, e, what)


def test_gradients_by_differences(device):
    """The loss sum(g y) is linear in each operand alone, so that a difference of two calls is its slope.

    Bars: both calls' outputs are off by what the module's bars say, and the slope by the gradient's."""
    gen = torch.Generator().manual_seed(6)
    x, base, down, up, ids, g = _make(150, 3, 40, 30, 6, torch.float32, gen, 10)
    ops = [x, down, up]
    grads = _run(device, x, base, down, up, ids, g, None)[1:]
    refs = _reference(x, base, down, up, ids, g, None)
    for i in range(3):
        v = torch.randn(ops[i].shape, generator=gen)
        hi, lo = list(ops), list(ops)
        hi[i], lo[i] = ops[i] + v, ops[i] - v
        change, bar = 0.0, 0.0
        for sign, o in ((1, hi), (-1, lo)):
            y = _run(device, o[0], base, o[1], o[2], ids, None, None)[0].double().cpu()
            (w, e), *_ = _reference(o[0], base, o[1], o[2], ids, None, None)
            change += sign * (g.double() * y).sum()
            bar += (g.double().abs() * (e + 3 * U32 * w.abs())).sum()
        step = hi[i].double() - lo[i].double()
        want = (grads[i].double().cpu() * step).sum()
        w, e = refs[1 + i]
        bar += ((e + 3 * U32 * w.abs()) * step.abs()).sum()
        assert (change - want).abs() <= bar, (i, change, want, bar)


@pytest.mark.parametrize("dtype", DTYPES, ids=lambda d: str(d)[6:])
def test_dropout_is_dropouts(device, dtype):
    """Dropping within the product is the product of what dropout leaves: with weights of one row and one entry, exactly."""
    gen = torch.Generator().manual_seed(7)
    N, H = 70, 36
    x = torch.randn(N, H, generator=gen).to(dtype).to(device)
    ids = torch.zeros(N, dtype=torch.long, device=device)
    kept = dropout(x, 0.5, seed=9, offset=2) != 0  # a scale of 2: exact products
    eye = torch.eye(H, device=device, dtype=dtype)
    for h in (0, 7, 8, 35):
        y = adapter_linear(x, eye[h].view(1, 1, H), torch.ones(1, 1, 1, device=device, dtype=dtype), ids, dropout_p=0.5,
                           seed=9, offset=2)
        assert torch.equal(y[:, 0], torch.where(kept[:, h], 2 * x[:, h], 0))
    # an offset on the device, and everything dropped
    at = torch.tensor([2], device=device)
    down, up = torch.randn(1, 4, H, device=device).to(dtype), torch.randn(1, 5, 4, device=device).to(dtype)
    a = adapter_linear(x, down, up, ids, dropout_p=0.5, seed=9, offset=at)
    assert torch.equal(a, adapter_linear(x, down, up, ids, dropout_p=0.5, seed=9, offset=2))
    xr = x.clone().requires_grad_()
    y = adapter_linear(xr, down, up, ids, dropout_p=1.0, seed=1)
    assert not y.any() and not torch.autograd.grad(y, xr, torch.ones_like(y))[0].any()


def test_float16_past_its_range(device):
    """t past 65504 in between, results within: float16's second product does not overflow."""
    N, H, O, r = 20, 64, 24, 3
    gen = torch.Generator().manual_seed(8)
    x = (torch.randn(N, H, generator=gen) * 3000).half()
    down = torch.randn(1, r, H, generator=gen).half() * 30
    up = (torch.randn(1, O, r, generator=gen) * 1e-4).half()
    ids = torch.zeros(N, dtype=torch.long)
    assert (x.double() @ down[0].double().T).abs().max() > 3e5
    g = (torch.randn(N, O, generator=gen) * 1e-3).half()
    out = _run(device, x, None, down, up, ids, g, torch.tensor([0.01]))
    want = _reference(x, None, down, up, ids, g, torch.tensor([0.01]))
    _close(out[0], want[0][0], want[0][1], "y")
    _close(out[1], want[1][0], want[1][1], "dx")


def test_values_that_are_no_numbers_stay_in_their_rows(device):
    """A NaN or an infinity in a row changes that row, its adapter's gradients, and nothing else."""
    gen = torch.Generator().manual_seed(9)
    for dtype in DTYPES:
        x, base, down, up, ids, g = _make(90, 3, 40, 32, 5, dtype, gen, 10, none=0.0)
        clean = _run(device, x, base, down, up, ids, g, None)
        bad = x.clone()
        bad[11, 3], bad[12, 0] = float("nan"), float("inf")
        out = _run(device, bad, base, down, up, ids, g, None)
        rows = torch.ones(90, dtype=torch.bool)
        rows[11] = rows[12] = False
        assert torch.isnan(out[0][11]).all() and not torch.isfinite(out[0][12]).any()
        assert torch.equal(out[0][rows.to(device)], clean[0][rows.to(device)])
        assert torch.equal(out[1], clean[1])
        others = [a for a in range(3) if a not in (int(ids[11]), int(ids[12]))]
        assert torch.equal(out[2][others], clean[2][others])
        # an infinite entry of up or down stays with its adapter
        up2 = up.clone()
        up2[1, 4, 2] = float("inf")
        out = _run(device, x, base, down, up2, ids, g, None)
        same = (ids != 1).to(device)
        assert torch.equal(out[0][same], clean[0][same]) and torch.equal(out[1][same], clean[1][same])


def test_strides(device):
    """Sliced, transposed, expanded and odd-addressed operands give what their copies give."""
    gen = torch.Generator().manual_seed(10)
    dtype = torch.bfloat16
    x, base, down, up, ids, g = (v.to(device) for v in _make(60, 3, 40, 32, 8, dtype, gen))
    want = adapter_linear(x, down, up, ids, base=base)
    wide = torch.zeros(60, 47, dtype=dtype, device=device)
    wide[:, 3:43] = x
    wb = torch.zeros(60, 35, dtype=dtype, device=device)
    wb[:, 1:33] = base
    wd = torch.zeros(3, 9, 45, dtype=dtype, device=device)
    wd[:, :8, 5:] = down
    wu = torch.zeros(3, 33, 11, dtype=dtype, device=device)
    wu[:, 1:, 3:] = up
    two = torch.stack([ids, ids], 1)[:, 0]
    got = adapter_linear(wide[:, 3:43], wd[:, :8, 5:], wu[:, 1:, 3:], two, base=wb[:, 1:33])
    assert torch.equal(got, want)
    got = adapter_linear(x.t().contiguous().t(), down.transpose(1, 2).contiguous().transpose(1, 2),
                         up.transpose(1, 2).contiguous().transpose(1, 2), ids, base=base.t().contiguous().t())
    assert torch.equal(got, want)
    got = adapter_linear(x.view(3, 20, 40), down, up, ids.view(3, 20), base=base.view(3, 20, 32))
    assert torch.equal(got.view(60, 32), want)
    # one row, factors and base expanded, and their gradients
    leaves = [v.clone().requires_grad_() for v in (x[:1], down[:1], up[:1], base[:1])]
    e = [leaves[0].expand(60, 40), leaves[1].expand(3, 8, 40), leaves[2].expand(3, 32, 8), leaves[3].expand(60, 32)]
    a = adapter_linear(e[0], e[1], e[2], ids, base=e[3])
    b = adapter_linear(e[0].contiguous(), e[1].contiguous(), e[2].contiguous(), ids, base=e[3].contiguous())
    assert torch.equal(a, b)
    ga, gb = torch.autograd.grad(a, leaves, g), torch.autograd.grad(b, leaves, g)
    for p, q in zip(ga, gb):
        assert torch.equal(p, q)
    # a gradient that is one number, expanded
    xr = x.clone().requires_grad_()
    (p,) = torch.autograd.grad(adapter_linear(xr, down, up, ids).float().sum(), xr)
    (q,) = torch.autograd.grad(adapter_linear(xr, down, up, ids), xr, torch.ones(60, 32, dtype=dtype, device=device))
    assert torch.equal(p, q)
    # one sequence [H] with one id
    v = adapter_linear(x[0], down, up, ids[0], base=base[0])
    assert v.shape == (32,) and torch.equal(v, want[0])


def test_empty(device):
    down, up = torch.randn(2, 4, 8, device=device), torch.randn(2, 6, 4, device=device)
    leaves = [torch.zeros(0, 8, device=device), down, up]
    for v in leaves:
        v.requires_grad_()
    y = adapter_linear(*leaves, torch.zeros(0, dtype=torch.long, device=device))
    assert y.shape == (0, 6)
    dx, dd, du = torch.autograd.grad(y, leaves, torch.zeros(0, 6, device=device))
    assert dx.shape == (0, 8) and not dd.any() and not du.any() and dd.shape == down.shape


def test_a_row_does_not_depend_on_the_batch(device):
    """A row's bits are the same alone, in any order and beside any others of its batch's size class."""
    gen = torch.Generator().manual_seed(11)
    for dtype in DTYPES:
        x, base, down, up, ids, _ = (v.to(device) for v in _make(1500, 5, 72, 56, 16, dtype, gen))
        want = adapter_linear(x, down, up, ids, base=base)
        order = torch.randperm(1500, generator=gen).to(device)
        assert torch.equal(adapter_linear(x[order], down, up, ids[order], base=base[order]), want[order])
        some = adapter_linear(x[:40], down, up, ids[:40], base=base[:40])
        assert torch.equal(adapter_linear(x[39:40], down, up, ids[39:40], base=base[39:40]), some[39:40])


def test_captured(device):
    """A captured step: forward and backward with an offset that moves, eager work between the replays."""
    gen = torch.Generator().manual_seed(12)
    x, base, down, up, ids, g = (v.to(device) for v in _make(400, 3, 64, 48, 8, torch.bfloat16, gen, 30))
    at = torch.zeros(1, dtype=torch.int64, device=device)

    def step(x, down, up, offset):
        leaves = [v.detach().requires_grad_() for v in (x, down, up)]
        y = adapter_linear(*leaves, ids, base=base, dropout_p=0.1, seed=3, offset=offset)
        return (y.detach(), *torch.autograd.grad(y, leaves, g))

    step(x, down, up, 0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(x, down, up, at)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(x, down, up, at)
        at.add_(1)
    for k in range(4):
        x.normal_()
        ids.copy_(ids.roll(37))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, step(x, down, up, k)):
            assert torch.equal(a, b)


def test_rollout_and_training_of_adapter_policies(device):
    """One step of three policies that share a model: tokens drawn from adapted logits, and the loss on them.

    The rollout's log-probs at temperature 1 are the trainer's recomputation on the same logits, so the ratio is 1;
    a policy's gradient comes from its own sequences alone."""
    gen = torch.Generator().manual_seed(13)
    B, T, H, V, A, r = 6, 9, 64, 1000, 3, 8
    hidden = torch.randn(B, T, H, generator=gen).to(torch.bfloat16).to(device)
    head = (torch.randn(V, H, generator=gen) * 0.2).to(torch.bfloat16).to(device)
    down = (torch.randn(A, r, H, generator=gen) * 0.1).to(torch.bfloat16).to(device).requires_grad_()
    up = (torch.randn(A, V, r, generator=gen) * 0.1).to(torch.bfloat16).to(device).requires_grad_()
    policy = torch.tensor([0, 1, 1, 0, 1, 0], device=device)[:, None].expand(B, T)
    logits = adapter_linear(hidden, down, up, policy, base=F.linear(hidden, head))
    u = torch.rand(B * T, generator=gen).to(device)
    out = sample_tokens(logits.detach().view(B * T, V), u)
    tokens, old = out.token_ids.view(B, T), out.logprobs.view(B, T)
    adv = torch.randn(B, 1, generator=gen).to(device).expand(B, T)
    mask = torch.ones(B, T, dtype=torch.bool, device=device)
    logp = R.gather_token_logprobs(logits, tokens)
    assert ((logp - old).abs() <= 1e-5 * old.abs() + 1e-6).all()
    loss = R.clipped_policy_loss(logp, old, adv, mask, clip_low=0.2, clip_high=0.2).loss
    dd, du = torch.autograd.grad(loss, (down, up))
    assert dd[:2].abs().sum(dim=(1, 2)).all() and not dd[2].any() and not du[2].any()
    # the same from the objective's own gradient of the logits
    leaf = logits.detach().requires_grad_()
    loss2 = R.clipped_policy_loss(R.gather_token_logprobs(leaf, tokens), old, adv, mask, clip_low=0.2, clip_high=0.2).loss
    (dl,) = torch.autograd.grad(loss2, leaf)
    _, _, want_d, want_u = _reference(hidden.view(-1, H).cpu(), None, down.detach().cpu(), up.detach().cpu(),
                                      policy.reshape(-1).cpu(), dl.view(-1, V).cpu(), None)
    _close(dd, *want_d, "ddown")
    _close(du, *want_u, "dup")


@pytest.mark.parametrize("N,A,r", [(300, 4096, 4), (1300, 4096, 3), (20, 4000, 128)])
def test_most_adapters(device, N, A, r):
    gen = torch.Generator().manual_seed(A)
    H, O = 24, 40
    x, base, down, up, ids, g = _make(N, A, H, O, r, torch.bfloat16, gen)
    ids[0], ids[1] = A - 1, 0
    out = _run(device, x, base, down, up, ids, g, None)
    want = _reference(x, base, down, up, ids, g, None)
    for got, (w, e), what in zip(out, want, ("y", "dx", "ddown", "dup")):
        _close(got, w, e, what)


@pytest.mark.parametrize("dtype,N,H,O,r", [(torch.bfloat16, 70000, 1024, 1088, 16), (torch.float32, 40000, 1000, 896, 9)],
                         ids=["bfloat16", "float32"])
def test_matrices_larger_than_the_caches(device, dtype, N, H, O, r):
    """Operands that are streamed, whole and not whole sizes: some rows, and the factors' gradients over all."""
    gen = torch.Generator(device="cuda").manual_seed(N)
    x, g, base = (torch.randn(N, c, generator=gen, device=device).to(dtype) for c in (H, O, O))
    down = (torch.randn(2, r, H, generator=gen, device=device) * H ** -0.5).to(dtype)
    up = torch.randn(2, O, r, generator=gen, device=device).to(dtype)
    ids = (torch.arange(N, device=device) // 5000) % 2
    ids[777:900] = -1
    leaves = [v.requires_grad_() for v in (x, down, up)]
    y = adapter_linear(*leaves, ids, base=base, dropout_p=0.1, seed=4)
    dx, dd, du = torch.autograd.grad(y, leaves, g)
    mask, factor = keep(N, H, 0.1, 4, 0)
    want = _reference(x.detach(), base, down.detach(), up.detach(), ids, g, None, mask.to(device), factor)
    some = torch.randint(0, N, (400,), generator=gen, device=device)
    some[:4] = torch.tensor([0, N - 1, 777, 4999], device=device)
    for got, (w, e), what in ((y[some], [v[some] for v in want[0]], "y"), (dx[some], [v[some] for v in want[1]], "dx"),
                              (dd, want[2], "ddown"), (du, want[3], "dup")):
        _close(got, w.cpu(), e.cpu(), what)


def test_two_threads(device):
    """Steps from two host threads on streams of their own give the bits of steps in turn."""
    import threading

    gen = torch.Generator().manual_seed(15)
    sets = [[v.to(device) for v in _make(600, 3, 80, 72, 12, torch.bfloat16, gen, 7)] for _ in range(2)]

    def step(x, base, down, up, ids, g):
        leaves = [v.detach().requires_grad_() for v in (x, down, up)]
        y = adapter_linear(*leaves, ids, base=base, dropout_p=0.1, seed=1)
        return (y.detach(), *torch.autograd.grad(y, leaves, g))

    want = [step(*s) for s in sets]
    torch.cuda.synchronize()
    bad = []

    def work(i):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            for _ in range(10):
                got = step(*sets[i])
                stream.synchronize()
                if not all(torch.equal(a, b) for a, b in zip(got, want[i])):
                    bad.append(i)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad


def test_without_a_graph(device):
    """A call that nothing differentiates gives the recorded call's bits; forward mode is refused."""
    gen = torch.Generator().manual_seed(16)
    for N in (5, 1200):
        x, base, down, up, ids, _ = (v.to(device) for v in _make(N, 3, 40, 48, 8, torch.float16, gen))
        kw = dict(base=base, dropout_p=0.2, seed=3)
        y = adapter_linear(x, down, up, ids, **kw)
        assert y.grad_fn is None
        for k in range(3):
            leaves = [x, down, up]
            leaves[k] = leaves[k].clone().requires_grad_()
            z = adapter_linear(*leaves, ids, **kw)
            assert z.grad_fn is not None and torch.equal(y, z)
            with torch.no_grad():
                z = adapter_linear(*leaves, ids, **kw)
            assert z.grad_fn is None and torch.equal(y, z)
        z = adapter_linear(x, down, up, ids, base=base.clone().requires_grad_(), dropout_p=0.2, seed=3)
        assert z.grad_fn is not None and torch.equal(y, z)
    import torch.autograd.forward_ad as fwd
    with fwd.dual_level(), pytest.raises((RuntimeError, NotImplementedError)):
        adapter_linear(fwd.make_dual(x, torch.ones_like(x)), down, up, ids)


def test_gradients_of_transposed_factors(device):
    """Factors that are kept transposed: the gradients are those of their copies."""
    gen = torch.Generator().manual_seed(17)
    for dtype in (torch.bfloat16, torch.float32):
        x, base, down, up, ids, g = (v.to(device) for v in _make(70, 3, 40, 32, 8, dtype, gen))
        scales = torch.tensor([0.5, 9.0, 2.0, 9.0, 1.5, 9.0], device=device)[::2]
        turned = [v.transpose(1, 2).contiguous().transpose(1, 2).requires_grad_() for v in (down, up)]
        plain = [v.clone().requires_grad_() for v in (down, up)]
        grads = []
        for d, u in (turned, plain):
            xr = x.clone().requires_grad_()
            y = adapter_linear(xr, d, u, ids, base=base, scales=scales, dropout_p=0.1, seed=2)
            grads.append(torch.autograd.grad(y, [xr, d, u], g))
        for p, q in zip(*grads):
            assert torch.equal(p, q)
