"""Drafts from the framework's own sampler, verified: the tokens that come out are
distributed as the target (MI355X).

The sampler draws from max(q, 1e-9), normalised: at most V 1e-9 of the mass away from
the q that verification is given, and the tokens' distribution by no more.  Shares over
B draws are within six standard deviations, sqrt(p (1 - p) / B) each.
"""

from __future__ import annotations

import math

import pytest
import torch

from rosellm_amd import roseinfer as RI

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("T", [1.0, 0.7])
@pytest.mark.parametrize("V", [5, 40])
def test_sampled_drafts_are_verified_to_the_targets_distribution(device, V, T, masked):
    g = torch.Generator().manual_seed(V)
    B, K = 80000, 2
    x = torch.randn(K + 1, V, generator=g) * 1.5
    y = x[:K] + torch.randn(K, V, generator=g)
    if masked:  # a filter on both sides
        x[:, ::3] = -math.inf
        y[:, ::3] = -math.inf
    x, y = x.expand(B, K + 1, V).to(device), y.expand(B, K, V).contiguous().to(device)
    d = torch.stack([RI.sample_next_token_batch(y[:, j].contiguous(), T, 0, 1.0, True, seed=V + 1, offset=j).token_ids
                     for j in range(K)], 1)
    u = torch.rand(B, K + 1, generator=g).to(device)
    out = RI.verify_draft_tokens(x, d, y, u, T)
    p = torch.softmax(x[0].double() / T, -1)
    for j in range(K):
        # position j's tokens, over the sequences that got that far: whether one did depends on its uniforms and
        # earlier drafts only
        tok = out.token_ids[out.num_accepted >= j, j]
        n = tok.numel()
        assert n > 1000
        freq = torch.bincount(tok, minlength=V).double() / n
        bar = 6 * (p[j] * (1 - p[j]) / n).sqrt() + V * 1e-9
        assert ((freq - p[j]).abs() <= bar).all(), (j, freq, p[j])
