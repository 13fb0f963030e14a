"""Log-probs of tokens from given uniforms where they are next to 0 (MI355X).

A row's only token has log-prob 0, exactly.  Elsewhere, with r the weight of what is left
beside the token, over the token's: the weights of both are within 2.2e-12 (two
polynomials of 1.1e-12 each), so -log1p(r) is off by at most 5e-12 of it, and by 1e-14
where a sum of 64-bit numbers is rounded (some forty additions of 2^-53 of the whole);
its rounding to float32 is 2^-24.
"""

from __future__ import annotations

import math

import pytest
import torch

from rosellm_amd.roseinfer import sample_tokens

from _sample_oracle import choose

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def _near(got, want):
    got, want = got.double().cpu(), torch.as_tensor(want, dtype=torch.float64)
    want = want.expand(got.shape)
    bar = (2.0 ** -24 + 5e-12) * want.abs() + 1e-14
    i = int(((got - want).abs() - bar).argmax())
    assert (got[i] - want[i]).abs() <= bar[i], (i, got[i].item(), want[i].item(), bar[i].item())


@pytest.mark.parametrize("dtype", DTYPES, ids=lambda d: str(d)[6:])
@pytest.mark.parametrize("V", [1, 9, 300, 8200, 151936])
def test_the_only_token_left_has_log_prob_0(device, V, dtype):
    gen = torch.Generator().manual_seed(V)
    B = 400 if V < 1000 else 60
    x = torch.randn(B, V, generator=gen) * 2.5
    at = torch.randint(0, V, (B,), generator=gen)
    x[torch.arange(B), at] = 20.0 + torch.rand(B, generator=gen) * 5
    x = x.to(dtype).to(device)
    u = torch.rand(B, generator=gen).to(device)
    T = (0.3 + torch.rand(B, generator=gen)).to(device)
    for kw in (dict(top_k=1), dict(top_p=1e-6), dict(min_p=1.0), dict(top_k=5, top_p=1e-6), dict(top_p=0.5, min_p=1.0)):
        for t in (0.8, T):
            out = sample_tokens(x, u, temperature=t, **kw)
            assert torch.equal(out.token_ids.cpu(), at)
            assert (out.sampling_logprobs == 0).all(), out.sampling_logprobs.min()
    # the only token that is possible at all
    x = torch.full_like(x, -math.inf).scatter_(1, at.to(device)[:, None], x.gather(1, at.to(device)[:, None]))
    for kw in (dict(), dict(top_k=3), dict(top_p=0.9), dict(min_p=0.1), dict(temperature=0.0)):
        out = sample_tokens(x, u, **{"temperature": T, **kw})
        assert torch.equal(out.token_ids.cpu(), at)
        assert (out.logprobs == 0).all() and (out.sampling_logprobs == 0).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=lambda d: str(d)[6:])
def test_a_token_beside_small_ones(device, dtype):
    """Two entries of which the second weighs down to 1e-13 of the first."""
    gen = torch.Generator().manual_seed(2)
    far = torch.linspace(0.5, 30.0, 60)
    x = torch.full((60, 500), -math.inf)
    m = torch.randn(60, generator=gen).to(dtype).float()
    x[:, 3], x[:, 400] = m, (m - far).to(dtype).float()
    gap = x[:, 3].double() - x[:, 400].double()
    for kw in (dict(), dict(top_k=2), dict(min_p=1e-15), dict(temperature=0.9)):
        T = kw.get("temperature", 1.0)
        out = sample_tokens(x.to(dtype).to(device), torch.full((60,), 0.25, device=device), **kw)
        assert (out.token_ids == 3).all()
        want = -torch.log1p(torch.exp(-gap / T))
        _near(out.logprobs, want)
        _near(out.sampling_logprobs, want)


@pytest.mark.parametrize("dtype", DTYPES, ids=lambda d: str(d)[6:])
@pytest.mark.parametrize("V,low", [(50257, -31.5), (151936, -31.5), (1 << 18, -31.5), (300001, -30.25), (1 << 20, -30.25)])
def test_flat_tails(device, V, low, dtype):
    """One entry and many that each weigh less than half a unit of the sums that decide tokens."""
    assert math.exp(low) < (2.0 ** -45 if V <= 1 << 18 else 2.0 ** -43)
    x = torch.full((2, V), low)
    x[0, 5], x[1, V // 2] = 0.0, 0.0
    x = x.to(dtype).to(device)
    u = torch.full((2,), 0.5, device=device)
    for kw, n in ((dict(), V), (dict(min_p=1e-20), V), (dict(top_k=V // 2 + 1), V // 2 + 1), (dict(top_k=7), 7)):
        print(f"[tail] V={V} {dtype} {kw}", flush=True)
        out = sample_tokens(x, u, **kw)
        assert out.token_ids.tolist() == [5, V // 2]
        _near(out.logprobs, -math.log1p((V - 1) * math.exp(low)))
        _near(out.sampling_logprobs, -math.log1p((n - 1) * math.exp(low)))
    # at another temperature, and greedy
    out = sample_tokens(x * 2, u, temperature=2.0)
    _near(out.logprobs, -math.log1p((V - 1) * math.exp(low)))
    out = sample_tokens(x, u, temperature=0.0)
    _near(out.logprobs, -math.log1p((V - 1) * math.exp(low)))


def test_log_probs_do_not_depend_on_the_batch(device):
    """The same bits in batches whose rows are cut into parts of other lengths."""
    gen = torch.Generator().manual_seed(4)
    for dtype in (torch.float32, torch.bfloat16):
        x = torch.randn(500, 30011, generator=gen)
        x[:, 17] += torch.linspace(0.0, 30.0, 500)
        x = x.to(dtype).to(device)
        u = torch.rand(500, generator=gen).to(device)
        for kw in (dict(), dict(top_p=0.9), dict(top_k=1000), dict(min_p=1e-3)):
            want = sample_tokens(x, u, **kw)
            for n in (1, 3, 499):
                for a, b in zip(sample_tokens(x[-n:], u[-n:], **kw), want):
                    assert torch.equal(a, b[-n:])
            many = sample_tokens(x.repeat(3, 1), u.repeat(3), **kw)
            for a, b in zip(many, want):
                assert torch.equal(a[1000:], b)


@pytest.mark.parametrize("V", [3, 64, 65, 127, 129, 511, 1023, 1024, 4097])
def test_short_rows_whose_entries_lie_far_apart(device, V):
    """Rows with fewer bins than others, the last of which takes most entries."""
    gen = torch.Generator().manual_seed(V)
    for dtype in DTYPES:
        x = (torch.randn(40, V, generator=gen) * torch.linspace(0.1, 60.0, 40)[:, None]).to(dtype)
        u = torch.rand(40, generator=gen)
        for kw in (dict(top_k=2), dict(top_k=V - 1, top_p=0.99), dict(top_p=0.9999), dict(top_k=V // 2 + 1, temperature=9.0),
                   dict(top_p=0.999, temperature=20.0, min_p=1e-5)):
            out = sample_tokens(x.to(device), u.to(device), **kw)
            for b in range(40):
                t, lp, lq = choose(x[b], u[b].item(), kw.get("temperature", 1.0), kw.get("top_k", 0), kw.get("top_p", 1.0),
                                   kw.get("min_p", 0.0))
                assert int(out.token_ids[b]) == t, (V, dtype, kw, b)
                _near(out.logprobs[b:b + 1], torch.tensor([lp], dtype=torch.float64))
                _near(out.sampling_logprobs[b:b + 1], torch.tensor([lq], dtype=torch.float64))
