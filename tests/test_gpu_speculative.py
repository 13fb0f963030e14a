"""Draft verification against a 64-bit restatement on the host (MI355X).

Tokens and counts have to be equal wherever the 64-bit result is decided: a
border (an acceptance ratio, a running sum) within 1e-9 of the whole of where
the uniform falls could go either way (the kernel's exponentials are good to
1.1e-12, its sums of at most 2^18 terms to 2^18 2^-53 = 3e-11), and the inputs'
seeds leave none.  Log-probs are float64 rounded once: 2^-24 relative, and 1e-11
absolute from the exponentials' and sums' error.
"""

from __future__ import annotations

import math

import pytest
import torch

from rosellm_amd import roseinfer as RI
from rosellm_amd.rosetrainer import embedding

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def _oracle(x, d, y, u, T, greedy):
    """(tokens, count, log-probs, decided) of one sequence."""
    K1, V = x.shape
    toks, lps = [-1] * K1, [0.0] * K1
    decided = True
    for j in range(K1):
        z = x[j].double()
        bad = bool((torch.isnan(z) | (z == math.inf)).any()) or bool((z == -math.inf).all())
        dj = int(d[j]) if j < K1 - 1 else -1
        drafted = dj >= 0
        if bad or dj >= V:
            lps[j] = math.nan
            return toks, j, lps, decided
        t = 1.0 if greedy else T
        z = z - z.max()
        e = torch.exp(z / t)
        p = e / e.sum()
        logp = lambda v: float(z[v] / t - torch.log(e.sum()))
        if greedy:
            best = int(z.argmax())
            if drafted and dj == best:
                toks[j], lps[j] = dj, logp(dj)
                continue
            toks[j], lps[j] = best, logp(best)
            return toks, j, lps, decided
        rest = p
        if drafted:
            if y is None:
                q = torch.zeros_like(p)
                q[dj] = 1.0
            else:
                w = y[j].double()
                if bool((torch.isnan(w) | (w == math.inf)).any()) or bool((w == -math.inf).all()):
                    lps[j] = math.nan
                    return toks, j, lps, decided
                q = torch.softmax((w - w.max()) / T, 0)
            uq = float(u[j]) * float(q[dj])
            decided &= abs(uq - float(p[dj])) > 1e-9 * max(uq, float(p[dj])) or uq == float(p[dj]) == 0.0
            if uq < float(p[dj]):
                toks[j], lps[j] = dj, logp(dj)
                continue
            rest = (p - q).clamp_min(0)
            if float(rest.sum()) <= 0:
                rest = p
            else:
                decided &= float(rest.sum()) > 1e-6  # else the difference itself is of few digits
        run = rest.cumsum(0)
        border = float(u[K1 - 1]) * float(run[-1])
        tok = int(torch.searchsorted(run, torch.tensor(border, dtype=torch.float64), right=True))
        near = run[max(tok - 1, 0):tok + 1]
        decided &= bool(((near - border).abs() > 1e-9 * float(run[-1])).all()) or border == 0.0
        toks[j], lps[j] = tok, logp(tok)
        return toks, j, lps, decided
    raise AssertionError


def _check(out, x, d, y, u, T=1.0, greedy=False, all_decided=True):
    tok, cnt, lp = out.token_ids.cpu(), out.num_accepted.cpu(), out.logprobs.double().cpu()
    x, d = x.cpu(), d.cpu()
    y, u = (None if v is None else v.cpu() for v in (y, u))
    assert out.logprobs.dtype == torch.float32 and tok.dtype == cnt.dtype == torch.int64
    for b in range(x.shape[0]):
        want = _oracle(x[b], d[b], None if y is None else y[b], None if u is None else u[b], T, greedy)
        if not want[3]:
            assert not all_decided, (b, "undecided")
            continue
        assert tok[b].tolist() == want[0], (b, tok[b].tolist(), want[0])
        assert int(cnt[b]) == want[1], b
        ref = torch.tensor(want[2], dtype=torch.float64)
        assert torch.equal(torch.isnan(ref), torch.isnan(lp[b])), b
        err = (lp[b] - ref).abs()
        assert (err <= 2 ** -24 * ref.abs() + 1e-11).logical_or(torch.isnan(ref)).all(), (b, err)


def _inputs(B, K, V, dtype, device, seed, ragged=False, noise=0.7, T=1.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(B, K + 1, V, generator=g) * 2.5
    x.scatter_add_(-1, torch.randint(0, V, (B, K + 1, 6), generator=g), 8 * torch.rand(B, K + 1, 6, generator=g))
    y = (x[:, :K] + noise * torch.randn(B, K, V, generator=g)).to(dtype)
    x = x.to(dtype)
    d = (y.float() / T - torch.log(-torch.log(torch.rand(B, K, V, generator=g).clamp_min(1e-30)))).argmax(-1)
    if ragged:
        d = d.masked_fill(torch.arange(K) >= torch.randint(0, K + 1, (B, 1), generator=g), -1)
    u = torch.rand(B, K + 1, generator=g)
    return [v.to(device) for v in (x, d, y, u)]


SIZES = [
    # B, K, V, T, ragged
    (1, 1, 1, 1.0, False),
    (3, 2, 2, 1.0, True),
    (5, 0, 100, 1.0, False),
    (8, 3, 7, 0.7, True),
    (4, 4, 4095, 1.0, False),
    (4, 4, 4096, 1.3, True),
    (4, 4, 4097, 1.0, False),
    (9, 5, 33333, 0.6, True),
    (2, 70, 1001, 1.0, True),
    (6, 4, 50257, 1.0, False),
    (4, 3, 151936, 0.9, True),
]


@pytest.mark.parametrize("with_q", [True, False])
@pytest.mark.parametrize("dtype", DTYPES, ids=lambda d: str(d)[6:])
@pytest.mark.parametrize("B,K,V,T,ragged", SIZES)
def test_verify(device, B, K, V, T, ragged, dtype, with_q):
    print(f"[verify] B={B} K={K} V={V} T={T} {dtype} q={with_q}", flush=True)
    x, d, y, u = _inputs(B, K, V, dtype, device, B + K + V, ragged, T=T)
    y = y if with_q else None
    out = RI.verify_draft_tokens(x, d, y, u, T)
    _check(out, x, d, y, u, T)
    again = RI.verify_draft_tokens(x, d.int(), y, u, T)
    assert all(torch.equal(p, q) for p, q in zip(out, again))


@pytest.mark.parametrize("dtype", DTYPES, ids=lambda d: str(d)[6:])
def test_verify_greedy(device, dtype):
    """First maxima, drafts that tie with them, and logits on a coarse grid; draft logits are not looked at."""
    g = torch.Generator().manual_seed(3)
    B, K, V = 12, 4, 9001
    x = torch.randint(-3, 4, (B, K + 1, V), generator=g).to(dtype)
    x[::2].scatter_(-1, torch.randint(0, V, (6, K + 1, 3), generator=g), 5.0)
    d = x[:, :K].float().argmax(-1)
    d[3, 1], d[4, 0], d[5, 2] = 8999, -1, int((x[5, 2] == x[5, 2].max()).nonzero()[-1])
    x, d = x.to(device), d.to(device)
    nan = torch.full((B, K, V), math.nan, dtype=dtype, device=device)
    for out in (RI.verify_draft_tokens(x, d, None, None, do_sample=False),
                RI.verify_draft_tokens(x, d, nan, None, -1.0)):
        _check(out, x, d, None, None, greedy=True)


def test_verify_extreme_uniforms(device):
    """0 takes every draft of any probability and the first entry of the rest, just under 1 the last."""
    x, d, y, _ = _inputs(6, 3, 5000, torch.float32, device, 31)
    x[:, :, :7] = -math.inf
    x[:, :, 4990:] = -math.inf
    y[:, :, 4980:] = -math.inf
    for v in (0.0, 1.0 - 2.0 ** -24, 0.5):
        u = torch.full((6, 4), v, device=device)
        for q in (y, None):
            _check(RI.verify_draft_tokens(x, d, q, u), x, d, q, u, all_decided=v == 0.5)
    u = torch.zeros(6, 4, device=device)
    out = RI.verify_draft_tokens(x, d, y, u)
    ok = torch.isfinite(x[:, :3].gather(-1, d[..., None])).all(1).flatten()
    assert torch.equal(out.num_accepted[ok], torch.full_like(out.num_accepted[ok], 3))
    assert (out.token_ids[ok, 3] == 7).all()
    u[:, 3] = 1.0 - 2.0 ** -24
    out = RI.verify_draft_tokens(x, d, y, u)
    assert (out.token_ids.max(1).values < 4990).all()


def test_verify_equal_rows_accept_everything(device):
    x, d, y, u = _inputs(4, 5, 20011, torch.bfloat16, device, 37)
    u[:, :5] = 1.0 - 2.0 ** -24
    out = RI.verify_draft_tokens(x, d, x[:, :5], u)
    assert (out.num_accepted == 5).all()
    _check(out, x, d, x[:, :5], u, all_decided=False)


def test_verify_masked_rows(device):
    """-inf and the type's lowest value as masks, one entry left, a draft that the mask or the draft model rules out."""
    for dtype in DTYPES:
        x, d, y, u = _inputs(8, 3, 4500, dtype, device, 41)
        low = torch.finfo(dtype).min
        keep = (torch.rand(4500, generator=torch.Generator().manual_seed(42)) < 0.3).to(device)
        keep[17] = True
        x[0:2, :, ~keep] = -math.inf
        x[2:4, :, ~keep] = low
        y[1:4, :, ~keep] = -math.inf
        x[4] = -math.inf
        x[4, :, 4321] = -3.0
        d[4, 0] = 4321
        x[5, 0, int(d[5, 0])] = -math.inf
        y[6, 0, int(d[6, 0])] = -math.inf
        x[7] = low
        for q in (y, None):
            _check(RI.verify_draft_tokens(x, d, q, u), x, d, q, u)


def test_verify_bad_rows(device):
    """NaN, +inf and empty rows and drafts of V or more end a sequence there; behind the end nothing is looked at."""
    x, d, y, u = _inputs(10, 3, 4500, torch.float32, device, 43)
    u[:, :3] = 1e-6  # drafts are accepted until something is wrong
    x[0, 0, 4400] = math.nan
    x[1, 1, 3] = math.inf
    x[2, 2] = -math.inf
    x[3, 3, 0] = math.nan
    y[4, 1, 77] = math.nan
    y[5, 0] = -math.inf
    d[6, 1] = 4500
    d[7, 2] = 2 ** 31 - 1
    d[8, 1] = -5
    d[8, 2] = 4500
    x[8, 2:] = math.nan
    y[8, 1:] = math.nan
    x[9, 1, 5] = math.inf
    u[9, 0] = 1.0 - 2.0 ** -24
    x[9, 0, int(d[9, 0])] = -20.0  # rejected before the bad row
    for q in (y, None):
        _check(RI.verify_draft_tokens(x, d, q, u), x, d, q, u)
    _check(RI.verify_draft_tokens(x, d, None, None, 0.0), x, d, None, None, greedy=True)


def test_verify_small_and_large_temperatures(device):
    x, d, y, u = _inputs(5, 2, 6000, torch.float32, device, 47)
    for T in (1e-310, 1e-30, 1e-3, 50.0, 1e30):
        _check(RI.verify_draft_tokens(x, d, y, u, T), x, d, y, u, max(T, 1e-290), all_decided=False)


def test_verify_empty_batch(device):
    out = RI.verify_draft_tokens(torch.zeros(0, 3, 9, device=device), torch.zeros(0, 2, dtype=torch.long, device=device),
                                 None, torch.zeros(0, 3, device=device))
    assert out.token_ids.shape == (0, 3) and out.num_accepted.shape == (0,) and out.logprobs.shape == (0, 3)


def test_verify_strides(device):
    """Rows at odd element offsets, a padded vocabulary, transposed, broadcast and non-contiguous operands."""
    g = torch.Generator().manual_seed(53)
    B, K, V = 4, 3, 4611
    for dtype in DTYPES:
        base = (torch.randn(K + 1, B, V + 13, generator=g) * 3).to(dtype).to(device)
        x = base[:, :, 3:V + 3].transpose(0, 1)
        y = base[:K, :, 5:V + 5].transpose(0, 1)
        d = torch.randint(0, V, (K, B), generator=g).to(device).t()
        u = torch.rand(K + 1, 2 * B, generator=g).to(device)[:, ::2].t()
        _check(RI.verify_draft_tokens(x, d, y, u), x, d, y, u)
        one = x[:1].expand(B, K + 1, V)
        col = x.transpose(1, 2).contiguous().transpose(1, 2)
        _check(RI.verify_draft_tokens(one, d, y, u), one, d, y, u)
        _check(RI.verify_draft_tokens(col, d, y, u), x, d, y, u)


def test_verify_distribution(device):
    """First tokens over many uniforms are distributed as the target, whatever the draft."""
    g = torch.Generator().manual_seed(59)
    V, B = 6, 60000
    x = (torch.randn(1, 2, V, generator=g) * 1.5).expand(B, 2, V).to(device)
    y = (torch.randn(1, 1, V, generator=g) * 1.5).expand(B, 1, V).to(device)
    q = torch.softmax(y[0, 0], 0).cpu()
    d = torch.multinomial(q, B, replacement=True, generator=g)[:, None].to(device)
    u = torch.rand(B, 2, generator=g).to(device)
    out = RI.verify_draft_tokens(x, d, y, u)
    freq = torch.bincount(out.token_ids[:, 0].cpu(), minlength=V).double() / B
    p = torch.softmax(x[0, 0].double().cpu(), 0)
    # six standard deviations of a share over B draws
    assert ((freq - p).abs() <= 6 * (p * (1 - p) / B).sqrt()).all(), (freq, p)


def test_verify_captured_and_on_streams(device):
    """A captured verification replayed on new inputs, beside eager calls on another stream."""
    x, d, y, u = _inputs(6, 4, 30000, torch.bfloat16, device, 61)
    RI.verify_draft_tokens(x, d, y, u)
    torch.cuda.synchronize()
    graph, other = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = RI.verify_draft_tokens(x, d, y, u)
    with torch.cuda.graph(other, pool=graph.pool()):
        out2 = RI.verify_draft_tokens(x, d, None, u)
    side = torch.cuda.Stream(device=device)
    for k in range(3):
        for dst, src in zip((x, d, y, u), _inputs(6, 4, 30000, torch.bfloat16, device, 62 + k, ragged=True)):
            dst.copy_(src)
        graph.replay()
        got = [t.clone() for t in out]
        other.replay()
        got2 = [t.clone() for t in out2]
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            want, want2 = RI.verify_draft_tokens(x, d, y, u), RI.verify_draft_tokens(x, d, None, u)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        assert all(torch.equal(a, b) for a, b in zip(got2, want2))
        _check(want, x, d, y, u)


def test_verified_tokens_are_embedded(device):
    """What follows in a rollout: the verified tokens' input rows, the places past them empty."""
    x, d, y, u = _inputs(7, 3, 5000, torch.bfloat16, device, 67)
    out = RI.verify_draft_tokens(x, d, y, u)
    w = torch.randn(5000, 64, generator=torch.Generator().manual_seed(68)).to(device)
    rows = embedding(out.token_ids, w, scale=8.0, padding_idx=-1)
    want = torch.where((out.token_ids >= 0)[..., None], w[out.token_ids.clamp_min(0)] * 8.0, 0.0)
    assert torch.equal(rows, want)
