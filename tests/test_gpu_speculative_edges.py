"""Draft verification at the edges of its contract (MI355X): the workspace of
greedy calls that are given draft logits, rows whose difference has no mass,
temperatures next to 0 over rows whose maximum is 0, log-probs of tokens that
hold all mass, and drafts behind whose end the buffers stop.

Tokens have to be those of the 64-bit definition wherever the uniform falls further
than 1e-9 of the whole from a border between two entries (the kernel's exponentials
are good to 1.1e-12, its sums of a few thousand terms to 1e-12); the inputs' seeds
leave no other.
"""

from __future__ import annotations

import math

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


def _draws(p, u):
    """The entries that an inverse-CDF draw from p [V] takes for the uniforms u [n]."""
    run = p.double().cumsum(0)
    border = u.double() * run[-1]
    at = torch.searchsorted(run, border, right=True)
    near = torch.stack([run[(at - 1).clamp_min(0)], run[at]]) - border
    assert (near.abs() > 1e-9 * run[-1]).all(), "an undecided uniform"
    return at


@pytest.mark.parametrize("with_infs", [False, True])
@pytest.mark.parametrize("shift", [0.0, 3.0])
@pytest.mark.parametrize("V", [5000, 40961])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=lambda d: str(d)[6:])
def test_verify_equal_rows_without_the_draft(device, dtype, V, shift, with_infs):
    """A draft without mass in two rows that are equal, or equal but for a constant: drawn from the target."""
    print(f"[verify] equal rows V={V} {dtype} shift={shift} infs={with_infs}", flush=True)
    g = torch.Generator().manual_seed(V)
    n = 300
    row = torch.randint(-32, 33, (V,), generator=g) / 8.0  # whole eighths up to 7: exact in every type
    row[17] = -math.inf
    if with_infs:
        row[torch.rand(V, generator=g) < 0.7] = -math.inf
    x = row.to(dtype).expand(n, 2, V).to(device)
    y = (row + shift).to(dtype).expand(n, 1, V).to(device)
    d = torch.full((n, 1), 17, device=device)
    u = torch.rand(n, 2, generator=g).to(device)
    out = RI.verify_draft_tokens(x, d, y, u)
    assert (out.num_accepted == 0).all()
    assert torch.equal(out.token_ids[:, 0], _draws(torch.softmax(x[0, 0].double(), 0), u[:, 1]))


def test_verify_small_difference_is_kept(device):
    """Rows that differ in one entry of 1e-12 of the mass only: it is all that the rest holds."""
    g = torch.Generator().manual_seed(5)
    n, V = 100, 5000
    row = torch.randn(V, generator=g)
    row[17] = row[4321] = -math.inf
    low = float(torch.logsumexp(row, 0)) - 27.6
    x = row.clone()
    x[4321] = low
    y = row.clone()
    y[17] = low
    d = torch.full((n, 1), 17, device=device)
    u = torch.rand(n, 2, generator=g).to(device)
    out = RI.verify_draft_tokens(x.expand(n, 2, V).to(device), d, y.expand(n, 1, V).to(device), u)
    assert (out.num_accepted == 0).all() and (out.token_ids[:, 0] == 4321).all()


@pytest.mark.parametrize("T", [1e-25, 1e-31, 1e-38, 1e-44, 1e-45, 3e-48, 1e-60, 1e-200, 1e-310])
def test_verify_small_temperatures_at_a_maximum_of_zero(device, T):
    """Log-probs and shifted logits have 0 as their maximum: all mass is at it, shared by its ties."""
    print(f"[verify] T={T}", flush=True)
    g = torch.Generator().manual_seed(7)
    B, K, V = 9, 2, 5003
    x = -torch.rand(B, K + 1, V, generator=g) - 0.5
    top = torch.randint(0, V, (B, K + 1), generator=g)
    x.scatter_(-1, top[..., None], 0.0)
    x[8, :, ::2] = -math.inf
    x[8].scatter_(-1, top[8][:, None], 0.0)
    x[5, 0, 4999], x[5, 0, 3] = 0.0, 0.0
    top[5, 0] = 3  # the first of the tied, which the uniform below takes
    y = -torch.rand(B, K, V, generator=g) - 0.5
    y.scatter_(-1, top[:, :K, None], 0.0)
    d = top[:, :K].clone()
    d[1, 1] = (d[1, 1] + 1) % V
    d[2, 0] = (d[2, 0] + 7) % V
    d[3, 0] = -1
    d[5, 0] = -1
    u = torch.rand(B, K + 1, generator=g).clamp(0.05, 0.95)
    u[5, K] = 0.2
    n = torch.tensor([2, 1, 0, 0, 2, 0, 2, 2, 2])
    for dtype in (torch.float32, torch.bfloat16):
        xd, dd, ud = x.to(dtype).to(device), d.to(device), u.to(device)
        for q in (y.to(dtype).to(device), None):
            out = RI.verify_draft_tokens(xd, dd, q, ud, T)
            assert torch.equal(out.num_accepted.cpu(), n), T
            for b in range(B):
                j = int(n[b])
                assert out.token_ids[b].tolist() == top[b, :j + 1].tolist() + [-1] * (K - j), (T, b)
            want = torch.zeros(B, K + 1)
            want[5, 0] = -math.log((x[5, 0] == 0).sum())
            # float64 rounded once, and 1e-11 from the exponentials and sums
            assert ((out.logprobs.cpu() - want).abs() <= 2.0 ** -24 * want.abs() + 1e-11).all()


@pytest.mark.parametrize("T", [1e-44, 1e-46])
def test_verify_subnormal_logits_at_small_temperatures(device, T):
    """Subnormal steps below a maximum of 0, in proportion to the temperature, weigh as anywhere else."""
    g = torch.Generator().manual_seed(11)
    V, n = 3001, 200
    step = 2.0 ** -149
    row = -step * torch.randint(0, 2000, (V,), generator=g).double()
    row[5] = 0.0
    x = row.float()
    assert torch.equal(x.double(), row)
    u = torch.rand(n, 1, generator=g)
    out = RI.verify_draft_tokens(x.expand(n, 1, V).to(device), torch.zeros(n, 0, dtype=torch.long, device=device), None,
                                 u.to(device), T)
    p = torch.softmax(row / T, 0)
    want = _draws(p, u[:, 0])
    assert torch.equal(out.token_ids[:, 0].cpu(), want)
    lp = torch.log_softmax(row / T, 0)[want]
    assert ((out.logprobs[:, 0].double().cpu() - lp).abs() <= 2.0 ** -24 * lp.abs() + 1e-11).all()


@pytest.mark.parametrize("do_sample", [True, False])
def test_verify_logprobs_are_at_most_zero(device, do_sample):
    """A token that holds all mass, or all but 1e-13 of it, whatever the logits' place."""
    g = torch.Generator().manual_seed(13)
    n, V = 400, 3000
    top = torch.randn(n, generator=g) * 10
    for rest in (-math.inf, 38.0):
        x = torch.full((n, 1, V), -math.inf) if rest < 0 else (top - rest)[:, None, None].expand(n, 1, V).clone()
        x[:, 0, 5] = top
        none = torch.zeros(n, 0, dtype=torch.long, device=device)
        out = RI.verify_draft_tokens(x.to(device), none, None, torch.full((n, 1), 0.5, device=device), do_sample=do_sample)
        assert (out.token_ids == 5).all()
        # 1e-11: the exponentials' and sums' error
        assert (out.logprobs <= 0).all() and (out.logprobs >= -1e-11).all()


@pytest.mark.parametrize("with_q", [True, False])
@pytest.mark.parametrize("B,K,V", [(1, 5, 151936), (7, 4, 5003), (3, 90, 1001), (2, 300, 130)])
def test_verify_rows_behind_the_last_end_need_not_exist(device, B, K, V, with_q):
    """The last sequence's draft is short and the operands stop with the rows it needs (what follows here is NaN);
    the sequences before it have drafts behind their ends that name entries."""
    print(f"[verify] short operands B={B} K={K} V={V} q={with_q}", flush=True)
    g = torch.Generator(device=device).manual_seed(B + K + V)
    x = torch.randn(B, K + 1, V, generator=g, device=device) * 2
    y = x[:, :K] + 0.3 * torch.randn(B, K, V, generator=g, device=device)
    d = torch.randint(0, V, (B, K), generator=g, device=device)
    d[:, :2] = y[:, :2].argmax(-1)
    d[:, 2] = -1
    d[-1, 1] = -1
    u = torch.rand(B, K + 1, generator=g, device=device) * 0.9
    want = RI.verify_draft_tokens(x, d, y if with_q else None, u)
    x.view(B * (K + 1), V)[(B - 1) * (K + 1) + 2:] = math.nan  # the last sequence's rows 0 and 1 are needed
    y.view(B * K, V)[(B - 1) * K + 1:] = math.nan              # and its draft's row 0
    got = _entry_point(x, d, y if with_q else None, u, 1.0, True)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert not torch.isnan(got[2]).any()
