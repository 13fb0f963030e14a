"""Draft verification at the edges of its contract (MI355X): the workspace of
greedy calls that are given draft logits."""

from __future__ import annotations

import pytest
import torch

from rosellm_amd import _native as nat
from rosellm_amd import roseinfer as RI

pytestmark = pytest.mark.gpu


def _entry_point(x, d, y, u, T, do_sample, size_of=None):
    """rrl_verify_drafts on contiguous operands, with a workspace of the promised size between guards."""
    B, K1, V = x.shape
    K = K1 - 1
    need = nat.lib().rrl_verify_drafts_workspace_bytes(*(size_of or (B, K, V, int(y is not None))))
    pad = 1 << 20
    room = torch.full((need + 2 * pad,), 0xA5, dtype=torch.uint8, device=x.device)
    tok = torch.full((B, K1), -7, dtype=torch.int64, device=x.device)
    cnt = torch.full((B,), -7, dtype=torch.int64, device=x.device)
    lp = torch.full((B, K1), 7.0, device=x.device)
    nat.call("rrl_verify_drafts", x.data_ptr(), nat.ptr(y), nat.dtype_code(x.dtype), B, K, V, K1 * V, V, K * V, V,
             nat.RrlView(d.data_ptr(), nat.I64, K, 1), nat.ptr(u), T, int(do_sample), tok.data_ptr(), cnt.data_ptr(),
             lp.data_ptr(), room.data_ptr() + pad, nat.stream_ptr(x.device))
    assert bool((room[:pad] == 0xA5).all()) and bool((room[pad + need:] == 0xA5).all())
    return tok, cnt, lp


# with and without the draft's rows these fall on both sides of a border between chunk sizes
@pytest.mark.parametrize("B,K,V", [(37, 1, 151936), (13, 4, 151936), (143, 4, 32000), (61, 2, 50257)])
def test_verify_greedy_with_draft_logits_stays_within_its_workspace(device, B, K, V):
    print(f"[verify] greedy B={B} K={K} V={V}", flush=True)
    g = torch.Generator(device=device).manual_seed(B + K)
    x = (torch.randn(B, K + 1, V, generator=g, device=device) * 2).to(torch.bfloat16)
    y = torch.randn(B, K, V, generator=g, device=device).to(torch.bfloat16)
    d = x[:, :K].float().argmax(-1)
    d[::3, K - 1] = 5
    u = torch.rand(B, K + 1, generator=g, device=device)
    want = RI.verify_draft_tokens(x, d, None, None, do_sample=False)
    for T, do_sample in ((1.0, False), (0.0, True)):
        got = _entry_point(x, d, y, u, T, do_sample)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    # and a workspace that was sized for a larger batch
    want = RI.verify_draft_tokens(x[:B // 2], d[:B // 2], y[:B // 2], u[:B // 2])
    got = _entry_point(x[:B // 2], d[:B // 2], y[:B // 2], u[:B // 2], 1.0, True, (B, K, V, 1))
    assert all(torch.equal(a, b) for a, b in zip(got, want))
