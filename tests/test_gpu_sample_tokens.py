"""Tokens from given uniforms with settings per row against 64-bit rows (MI355X).

Tokens are equal: a border lies within the kernel's 1e-11 of a running sum in one of some
million rows, and none of these.  Log-probs are rounded to float32 from numbers that are
within 2e-11 (ten errors of 1.1e-12 of an exponential, and sums to 1e-11), so |err| <=
2^-24 |ref| + 1e-10.
"""

from __future__ import annotations

import math

import pytest
import torch

from rosellm_amd.roseinfer import sample_tokens, verify_draft_tokens

from _sample_oracle import choose

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def _check(x, u, device, view=None, **kw):
    B = x.shape[0]
    dev = {k: v.to(device) if torch.is_tensor(v) else v for k, v in kw.items()}
    xd = x.to(device) if view is None else view
    out = sample_tokens(xd, u.to(device), **dev)
    def at(name, b, default):
        v = kw.get(name, default)
        return v[b].item() if torch.is_tensor(v) else v
    for b in range(B):
        t, lp, lq = choose(x[b], u[b].item(), at("temperature", b, 1.0), at("top_k", b, 0), at("top_p", b, 1.0),
                           at("min_p", b, 0.0))
        got = int(out.token_ids[b]), float(out.logprobs[b]), float(out.sampling_logprobs[b])
        assert got[0] == t, (b, got, t, lp)
        for g, w in ((got[1], lp), (got[2], lq)):
            assert (math.isnan(g) and math.isnan(w)) or abs(g - w) <= 2.0 ** -24 * abs(w) + 1e-10, (b, g, w)
        assert not got[1] > 0 and not got[2] > 0
    return out


def _logits(B, V, gen, dtype, kind):
    if kind == "ties":  # few values, so that cuts fall among equal entries
        return torch.randint(-3, 4, (B, V), generator=gen).to(dtype)
    if kind == "peaked":
        x = torch.randn(B, V, generator=gen)
        x[:, V // 3] += 14
        return x.to(dtype)
    if kind == "masked":  # most entries impossible, some at the type's lowest value
        x = torch.randn(B, V, generator=gen) * 3
        x = x.masked_fill(torch.rand(B, V, generator=gen) < 0.9, -math.inf)
        x[:, V // 2] = 1.0
        x = x.to(dtype)
        return torch.where(torch.rand(B, V, generator=gen) < 0.02, torch.finfo(dtype).min, x)
    return (torch.randn(B, V, generator=gen) * 2.5).to(dtype)


SETTINGS = [
    dict(),
    dict(temperature=0.7),
    dict(temperature=1.3, top_k=5),
    dict(top_p=0.9),
    dict(top_p=0.3, temperature=2.0),
    dict(min_p=0.05),
    dict(top_k=40, top_p=0.8, min_p=0.01, temperature=0.9),
    dict(temperature=0.0, top_k=3, top_p=0.5),
    dict(top_k=1),
    dict(top_p=1e-6),
    dict(min_p=1.0),
]
SIZES = [1, 2, 7, 8, 63, 65, 1000, 8191, 8193, 50257]


@pytest.mark.parametrize("dtype", DTYPES, ids=lambda d: str(d)[6:])
@pytest.mark.parametrize("V", SIZES)
def test_settings(device, V, dtype):
    gen = torch.Generator().manual_seed(V)
    for kind in ("normal", "ties", "peaked", "masked"):
        x = _logits(3, V, gen, dtype, kind)
        for kw in SETTINGS:
            print(f"[sample] V={V} {dtype} {kind} {kw}", flush=True)
            _check(x, torch.rand(3, generator=gen), device, **kw)


def _mixed(B, gen):
    def pick(values, dtype):
        return torch.tensor(values, dtype=dtype)[torch.randint(0, len(values), (B,), generator=gen)]

    return dict(temperature=pick([0.0, -1.0, 0.3, 0.8, 1.0, 1.7], torch.float32),
                top_k=pick([-1, 0, 0, 1, 20, 700, 10 ** 6], torch.int32),
                top_p=pick([0.0, 1.0, 1.5, 0.5, 0.9, 0.99], torch.float32),
                min_p=pick([-0.5, 0.0, 0.0, 0.01, 0.2, 2.0], torch.float32))


@pytest.mark.parametrize("dtype", DTYPES, ids=lambda d: str(d)[6:])
@pytest.mark.parametrize("B,V", [(300, 1003), (40, 32000), (24, 151936)])
def test_settings_of_their_own_for_every_row(device, B, V, dtype):
    gen = torch.Generator().manual_seed(B)
    x = torch.cat([_logits(B // 4, V, gen, dtype, kind) for kind in ("normal", "ties", "peaked", "masked")])
    kw = _mixed(x.shape[0], gen)
    u = torch.rand(x.shape[0], generator=gen)
    out = _check(x, u, device, **kw)
    # the same bits again, and with int64 top_k
    kw = {k: v.to(device) for k, v in kw.items()}
    again = sample_tokens(x.to(device), u.to(device), **{**kw, "top_k": kw["top_k"].long()})
    for a, b in zip(out, again):
        assert torch.equal(a, b)
    # without the sampling log-probs the rest is the same
    less = sample_tokens(x.to(device), u.to(device), **kw, sampling_logprobs=False)
    assert less.sampling_logprobs is None and torch.equal(less.token_ids, out.token_ids)
    # a row alone
    i = x.shape[0] // 2
    one = sample_tokens(x[i:i + 1].to(device), u[i:i + 1].to(device), **{k: v[i:i + 1] for k, v in kw.items()})
    assert torch.equal(one.token_ids, out.token_ids[i:i + 1])


@pytest.mark.parametrize("V", [300001, 1 << 20])
def test_long_rows(device, V):
    """Rows of more parts than others, of which the longer has fewer bits to a weight."""
    gen = torch.Generator().manual_seed(1)
    for dtype in (torch.float32, torch.bfloat16):
        x = _logits(2, V, gen, dtype, "normal")
        for kw in (dict(), dict(top_p=0.9), dict(top_k=3000), dict(top_k=100000, top_p=0.7, min_p=1e-4)):
            print(f"[sample] V={V} {dtype} {kw}", flush=True)
            _check(x, torch.rand(2, generator=gen), device, **kw)


def test_equal_entries(device):
    """Rows of one value: a cut among all of them, by place; and by exact shares."""
    for V in (4, 64, 4096, 16384):
        x = torch.zeros(4, V)
        x[1] = -7.5
        x[2] = 60000.0
        x[3] = torch.finfo(torch.float32).min
        for kw in (dict(top_k=V // 4), dict(top_p=0.5), dict(top_p=0.75, top_k=V // 2), dict(min_p=1.0)):
            for u in (0.0, 0.3, 0.9999999):
                _check(x, torch.full((4,), u), device, **kw)
    # zeros of both signs are equal
    x = torch.tensor([[0.0, -0.0, 0.0, -0.0, -1.0]])
    for u in (0.1, 0.4, 0.6, 0.9):
        out = _check(x, torch.tensor([u]), device, top_k=2)
        assert int(out.token_ids) < 2
        _check(x, torch.tensor([u]), device, min_p=1.0)
        _check(x.abs() * -1, torch.tensor([u]), device, min_p=1.0)


def test_uniforms_at_the_ends(device):
    x = torch.full((1, 5000), -math.inf)
    x[0, 100] = -600.0  # has a weight, of less than a unit
    x[0, 200] = 0.0
    x[0, 4000] = 1.0
    x[0, 4500] = -2000.0  # has none
    x[0, 50] = -2000.0
    u = torch.tensor([0.0])
    assert int(sample_tokens(x.to(device), u.to(device)).token_ids) == 100
    assert int(sample_tokens(x.to(device), u.to(device), top_k=2).token_ids) == 200
    for top in (1.0, 1.0 - 2.0 ** -24):
        assert int(sample_tokens(x.to(device), torch.tensor([top], device=device)).token_ids) == 4000
    # outside [0, 1): as the nearest end
    for bad, want in ((-1.0, 100), (math.nan, 100), (5.0, 4000)):
        assert int(sample_tokens(x.to(device), torch.tensor([bad], device=device)).token_ids) == want
    gen = torch.Generator().manual_seed(3)
    x = torch.randn(64, 9000, generator=gen)
    _check(x, torch.full((64,), 2.0 ** -24), device, top_p=0.9)
    _check(x, torch.full((64,), 1 - 2.0 ** -24), device, top_p=0.9)


def test_extreme_temperatures_and_values(device):
    gen = torch.Generator().manual_seed(6)
    x = torch.randn(2, 3000, generator=gen)
    u = torch.rand(2, generator=gen)
    for T in (1e-30, 1e-45, 1e-3, 1e3, 1e30, 3e38):
        for kw in (dict(), dict(top_k=7), dict(top_p=0.6), dict(min_p=0.3)):
            _check(x, u, device, temperature=T, **kw)
            _check(x, u, device, temperature=torch.full((2,), T), **kw)
    big = x * 1e37
    for kw in (dict(), dict(top_k=7), dict(top_p=0.6), dict(min_p=0.3), dict(temperature=1e37, top_p=0.5)):
        _check(big, u, device, **kw)
        _check(big.to(torch.bfloat16), u, device, **kw)
    _check(x * 1e-40, u, device, top_k=3)
    _check((x * 20000).clamp(-65504, 65504).to(torch.float16), u, device, top_p=0.9)


def test_rows_without_a_distribution(device):
    x = torch.randn(7, 700)
    x[0, 5] = math.nan
    x[1, 699] = math.inf
    x[2] = -math.inf
    T = torch.ones(7)
    T[3], T[4] = math.nan, math.inf
    for dtype in DTYPES:
        for kw in (dict(), dict(top_p=0.5), dict(top_k=5)):
            out = _check(x.to(dtype), torch.rand(7), device, temperature=T, **kw)
            assert (out.token_ids[:5] == -1).all() and (out.token_ids[5:] >= 0).all()
    out = sample_tokens(x.to(device), torch.rand(7, device=device), temperature=0.0)
    assert (out.token_ids[:3] == -1).all() and torch.isnan(out.logprobs[:3]).all()
    # settings that are NaN filter nothing
    nan = torch.full((7,), math.nan, device=device)
    y, u = torch.randn(7, 300, device=device), torch.rand(7, device=device)
    assert torch.equal(sample_tokens(y, u, top_p=nan, min_p=nan).token_ids, sample_tokens(y, u).token_ids)


def test_strides_and_empty(device):
    gen = torch.Generator().manual_seed(7)
    big = _logits(6, 9100, gen, torch.bfloat16, "normal").to(device)
    u = torch.rand(6, generator=gen)
    for v in (big[:, 1:9000], big[:, 3:], big[::2], big[:1].expand(4, 9100), big.t()[:6, :].contiguous().t()[:, :6],
              big[:, ::3]):
        _check(v.cpu(), u[:v.shape[0]], device, view=v, top_p=0.9, top_k=torch.full((v.shape[0],), 100))
    e = sample_tokens(big[:0], u[:0].to(device), top_k=torch.zeros(0, dtype=torch.int64, device=device))
    assert e.token_ids.shape == (0,)
    settings = torch.tensor([[0.7, 9.0], [1.2, 9.0]], device=device)[:, 0]  # a column
    two = torch.tensor([0.7, 1.2])
    a = sample_tokens(big[:2], u[:2].to(device), temperature=settings)
    b = sample_tokens(big[:2], u[:2].to(device), temperature=two.to(device))
    assert torch.equal(a.token_ids, b.token_ids)


def test_captured_and_on_a_stream(device):
    """Replays with new logits, settings and uniforms against eager calls, eager work between them."""
    gen = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(12, 20000, generator=gen, device=device)
    u = torch.rand(12, generator=gen, device=device)
    T = torch.ones(12, device=device)
    sample_tokens(x, u, temperature=T, top_p=0.9, top_k=500)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = sample_tokens(x, u, temperature=T, top_p=0.9, top_k=500)
    for k in range(4):
        x.normal_(generator=gen)
        u.uniform_(generator=gen)
        T.fill_(0.5 + 0.3 * k)
        graph.replay()
        torch.cuda.synchronize()
        want = sample_tokens(x, u, temperature=T, top_p=0.9, top_k=500)
        assert torch.equal(out.token_ids, want.token_ids) and torch.equal(out.logprobs, want.logprobs)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = sample_tokens(x, u, temperature=T, top_p=0.9, top_k=500)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got.token_ids, want.token_ids)


def test_frequencies(device):
    """Even uniforms give every token its share: V tokens, n uniforms (i + 1/2) / n, counts within one of n q."""
    gen = torch.Generator().manual_seed(2)
    x = torch.randn(1, 50, generator=gen)
    n = 20000
    u = (torch.arange(n) + 0.5) / n
    out = sample_tokens(x.to(device).expand(n, 50), u.to(device), top_k=20, top_p=0.9, temperature=0.8)
    z = x[0].double() / 0.8
    p, at = torch.sort(z.exp(), descending=True)
    p = p[:20] / p[:20].sum()
    m = max(1, int((p.cumsum(0) <= 0.9).sum()))
    q = torch.zeros(50, dtype=torch.float64)
    q[at[:m]] = p[:m] / p[:m].sum()
    counts = torch.bincount(out.token_ids.cpu(), minlength=50).double()
    # float32 uniforms are off by 2^-25: less than one count
    assert ((counts - n * q).abs() <= 1.01).all()


def test_drafts_drawn_by_it_are_verified(device):
    """Draft tokens drawn with the filter on both sides: drafts equal to the target are all accepted, with the same log-probs."""
    gen = torch.Generator().manual_seed(8)
    B, K, V = 5, 3, 4000
    x = (torch.randn(B, K + 1, V, generator=gen) * 3).to(device)
    u = torch.rand(B, K + 1, generator=gen).to(device)
    drafts = torch.stack([sample_tokens(x[:, j], u[:, j], temperature=0.8).token_ids for j in range(K)], 1)
    out = verify_draft_tokens(x, drafts, x[:, :K].contiguous(), u, 0.8)
    assert (out.num_accepted == K).all()
    last = sample_tokens(x[:, K], u[:, K], temperature=0.8)
    assert torch.equal(out.token_ids[:, K], last.token_ids)
    assert torch.equal(out.token_ids[:, :K], drafts)
    assert ((out.logprobs[:, K] - last.logprobs).abs() <= 2.0 ** -23 * last.logprobs.abs()).all()


@pytest.mark.parametrize("B,V", [(1100, 70001), (3000, 9), (700, 16385)])
def test_large_batches(device, B, V):
    """Longer parts where there are rows enough: some rows against 64 bits, all against calls of fewer rows."""
    gen = torch.Generator().manual_seed(B)
    x = _logits(B, V, gen, torch.bfloat16, "normal")
    kw = _mixed(B, gen)
    u = torch.rand(B, generator=gen)
    xd, ud, kd = x.to(device), u.to(device), {k: v.to(device) for k, v in kw.items()}
    whole = sample_tokens(xd, ud, **kd)
    for i in range(0, B, B // 3):
        n = min(B, i + 40)
        some = sample_tokens(xd[i:n], ud[i:n], **{k: v[i:n] for k, v in kd.items()})
        for a, b in zip(some, whole):
            assert torch.equal(a, b[i:n])
    pick = torch.arange(0, B, max(1, B // 8))
    _check(x[pick], u[pick], device, **{k: v[pick] for k, v in kw.items()})


def test_two_threads(device):
    """Calls from two host threads on streams of their own give the bits of calls in turn."""
    import threading

    gen = torch.Generator().manual_seed(5)
    xs = [_logits(20, 30000, gen, torch.bfloat16, "normal").to(device) for _ in range(2)]
    u = torch.rand(20, generator=gen).to(device)
    want = [sample_tokens(x, u, top_k=300, top_p=0.9) for x in xs]
    torch.cuda.synchronize()
    bad = []

    def work(i):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            for _ in range(10):
                got = sample_tokens(xs[i], u, top_k=300, top_p=0.9)
                stream.synchronize()
                if not (torch.equal(got.token_ids, want[i].token_ids) and torch.equal(got.logprobs, want[i].logprobs)):
                    bad.append(i)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad
