"""Log-probs of tokens from given uniforms where they are next to 0 (MI355X)."""

from __future__ import annotations

import math

import pytest
import torch

from rosellm_amd.roseinfer import sample_tokens

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]


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
