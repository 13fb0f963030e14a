"""Microscaled 4-bit blocks and their product against plain restatements (MI355X).

Codes and scales are whole numbers and have to be equal.  The product sums the
4-bit numbers' exact products in float32: with n = cols terms of which the
matrix unit may add 128 in any order, |err| <= n 2^-23 sum|x w| (one rounding to
2^-23 at most a term, truncation included), plus half a step of the output type.
"""

from __future__ import annotations

import math

import pytest
import torch

from rosellm_amd import _native as nat
from rosellm_amd import roseinfer as RI

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]
GRID = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)


def _quantize(x):
    """(codes, scales) of x [R, H], in 64 bits on the host."""
    R, H = x.shape
    P = (H + 127) // 128 * 128
    v = torch.zeros(R, P, dtype=torch.float64)
    v[:, :H] = x.double().cpu()
    v = v.view(R, P // 32, 32)
    amax = v.abs().amax(-1)
    bad = ~torch.isfinite(v).all(-1)
    amax = torch.where(bad, 1.0, amax)
    e = torch.frexp(amax).exponent.long() - 3
    e = torch.where(amax > 0, e, -127).clamp_min(-127)
    a = v.abs() / torch.ldexp(torch.ones_like(amax), e)[..., None]
    a = torch.where(bad[..., None], 0.0, a)
    up = torch.searchsorted(GRID, a.contiguous()).clamp_max(7)
    down = (up - 1).clamp_min(0)
    dist = (GRID[up] - a) - (a - GRID[down])
    code = torch.where((dist < 0) | ((dist == 0) & (up % 2 == 0)), up, down)
    code = code + 8 * torch.signbit(v).long()
    code = torch.where(bad[..., None], 0, code).view(R, P // 2, 2)
    return (code[..., 0] + 16 * code[..., 1]).to(torch.uint8), torch.where(bad, 255, e + 127).to(torch.uint8)


def _values(q):
    """The numbers that the blocks stand for, in 64 bits on the host."""
    codes, scales = q.codes.cpu().long(), q.scales.cpu().long()
    code = torch.stack([codes & 15, codes >> 4], -1).view(codes.shape[0], 2 * codes.shape[1])
    v = GRID[code & 7] * torch.where(code >= 8, -1.0, 1.0)
    unit = torch.ldexp(torch.ones(scales.shape, dtype=torch.float64), scales - 127)
    unit = torch.where(scales == 255, math.nan, unit)
    return (v.view(*scales.shape, 32) * unit[..., None]).view(code.shape)[:, :q.cols]


def _check_codes(q, x):
    codes, scales = _quantize(x)
    assert q.cols == x.shape[1]
    assert torch.equal(q.scales.cpu(), scales)
    assert torch.equal(q.codes.cpu(), codes)


@pytest.mark.parametrize("dtype", DTYPES, ids=lambda d: str(d)[6:])
@pytest.mark.parametrize("R,H", [(1, 1), (1, 31), (3, 32), (5, 33), (2, 127), (7, 128), (4, 129), (64, 1000),
                                 (33, 1024), (3, 4100)])
def test_quantize(device, R, H, dtype):
    g = torch.Generator().manual_seed(R + H)
    x = (torch.randn(R, H, generator=g) * torch.exp(4 * torch.randn(R, 1, generator=g))).to(dtype).to(device)
    q = RI.quantize_mxfp4(x)
    _check_codes(q, x)
    for t in DTYPES[:2]:
        got = RI.dequantize_mxfp4(q, t)
        assert got.shape == (R, H) and got.dtype == t
        assert torch.equal(got.double().cpu(), _values(q))
    assert torch.equal(RI.dequantize_mxfp4(q, torch.float16).cpu(), _values(q).to(torch.float16))


def test_quantize_every_bfloat16(device):
    """Every bfloat16 under block maxima from the smallest to the largest exponent, infinities and NaN among them."""
    every = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(torch.bfloat16)
    rows = []
    for e in range(0, 256, 3):
        top = torch.tensor((e << 7) | 93, dtype=torch.int16).view(torch.bfloat16)
        x = every.view(-1, 16)
        keep = x.abs().float() <= top.float().abs()
        x = torch.where(keep, x, torch.zeros_like(x))
        rows.append(torch.cat([x, top.expand(x.shape[0], 1), torch.zeros(x.shape[0], 15, dtype=x.dtype)], 1).view(-1, 1024))
    x = torch.cat(rows + [every.view(-1, 1024)])
    q = RI.quantize_mxfp4(x.to(device))
    _check_codes(q, x)
    back = RI.dequantize_mxfp4(q).double().cpu()
    want = _values(q)
    assert torch.equal(torch.isnan(back), torch.isnan(want))
    assert torch.equal(back.nan_to_num(), want.nan_to_num())


def test_quantize_borders(device):
    """Halfway points and their neighbours, subnormal and largest float32 blocks, signed zeros."""
    mid = torch.tensor([0.0, -0.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 7.0, 7.9999995])
    v = torch.cat([mid, torch.nextafter(mid, torch.tensor(9.0)), torch.nextafter(mid, torch.tensor(-9.0))])
    v = torch.cat([v[v < 8], -v[v < 8]])
    rows = []
    for e in (-149, -140, -130, -127, -126, -125, -100, -1, 0, 50, 100, 124, 125):
        for i in range(0, v.numel(), 30):
            part = v[i:i + 30]
            row = torch.zeros(32)
            row[:part.numel()] = torch.ldexp(part, torch.tensor(e))
            row[31] = torch.ldexp(torch.tensor(4.0), torch.tensor(min(e, 125)))
            rows.append(row)
    x = torch.stack(rows)
    x = x[torch.isfinite(x).all(1)]
    _check_codes(RI.quantize_mxfp4(x.to(device)), x)


def test_quantize_strides(device):
    g = torch.Generator().manual_seed(3)
    base = torch.randn(40, 301, generator=g)
    for dtype in DTYPES:
        b = base.to(dtype).to(device)
        for x in (b[:, 1:290], b[::3, 8:200], b.t(), b[:1].expand(6, 301), b[:, ::2], b[5:5]):
            _check_codes(RI.quantize_mxfp4(x), x)


def _check_linear(out, x, q):
    xq = RI.MxFp4(*_quantize(x.reshape(-1, x.shape[-1])), x.shape[-1])
    a, w = _values(xq), _values(q)
    want, mass = a @ w.t(), a.abs() @ w.abs().t()
    got = out.reshape(want.shape).double().cpu()
    f = torch.finfo(out.dtype)
    half = 0.0 if out.dtype == torch.float32 else f.eps / 2
    bar = x.shape[-1] * 2.0 ** -23 * mass * (1 + half) + half * want.abs() + f.smallest_normal * f.eps / 2
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    bad = (got - want).abs() > bar
    assert not bad.any(), (bad.nonzero()[:5], got[bad][:5], want[bad][:5])


SIZES = [
    # M, N, H
    (1, 1, 1),
    (1, 17, 32),
    (2, 5, 100),
    (3, 300, 128),
    (16, 1000, 256),
    (17, 64, 640),
    (31, 129, 96),
    (64, 515, 512),
    (65, 257, 1000),
    (130, 4097, 520),
    (300, 777, 2080),
    (40, 264, 500),
    (83, 520, 1024),
    (90, 1000, 1100),
    (150, 128, 130),
    (200, 2008, 900),
    (1, 151936, 64),
]


@pytest.mark.parametrize("dtype", DTYPES, ids=lambda d: str(d)[6:])
@pytest.mark.parametrize("M,N,H", SIZES)
def test_linear(device, M, N, H, dtype):
    print(f"[mxfp4] M={M} N={N} H={H} {dtype}", flush=True)
    g = torch.Generator().manual_seed(M + N + H)
    x = (torch.randn(M, H, generator=g) * torch.exp(torch.randn(1, H, generator=g))).to(dtype).to(device)
    w = (torch.randn(N, H, generator=g) * 0.05).to(dtype).to(device)
    q = RI.quantize_mxfp4(w)
    for out_dtype in (None, torch.float32):
        out = RI.mxfp4_linear(x, q, out_dtype)
        assert out.shape == (M, N) and out.dtype == (out_dtype or dtype)
        _check_linear(out, x, q)
    assert torch.equal(RI.mxfp4_linear(x, q, torch.float32), out)


def _guarded(rows, cols, dtype, device):
    """An [rows, cols] view in the middle of a buffer of a pattern, and a check that the rest still holds it."""
    pad = 4096
    base = torch.full((rows * cols + 2 * pad,), 77.0, dtype=dtype, device=device)
    return base[pad:pad + rows * cols].view(rows, cols), lambda: bool((base[:pad] == 77).all()
                                                                       and (base[pad + rows * cols:] == 77).all())


@pytest.mark.parametrize("M,N,H", [(2, 8, 64), (17, 264, 128), (65, 512, 640), (130, 1000, 1000), (250, 136, 1500),
                                   (1100, 60000, 70), (1100, 60008, 640), (1100, 60000, 1100), (5, 1 << 20, 96),
                                   (20, (1 << 20) + 8, 600), (9, 1 << 20, 1030), (33, 1 << 20, 40)])
def test_linear_stays_within_its_output(device, M, N, H):
    """Partial tiles of whole vectors and the wide slabs: the right values, and nothing beside them."""
    g = torch.Generator(device=device).manual_seed(M + N + H)
    x = torch.randn(M, H, generator=g, device=device).to(torch.bfloat16)
    q = RI.quantize_mxfp4(torch.randn(N, H, generator=g, device=device).to(torch.bfloat16))
    lib = nat.lib()
    for dtype, code in ((torch.bfloat16, nat.BF16), (torch.float32, nat.F32)):
        out, intact = _guarded(M, N, dtype, device)
        ws = torch.full((lib.rrl_mxfp4_linear_workspace_bytes(M, H),), 255, dtype=torch.uint8, device=device)
        nat.call("rrl_mxfp4_linear", x.data_ptr(), nat.BF16, M, H, H, q.codes.data_ptr(), q.scales.data_ptr(), N,
                 out.data_ptr(), code, ws.data_ptr(), nat.stream_ptr(x.device))
        assert intact()
        a = RI.dequantize_mxfp4(RI.quantize_mxfp4(x)).double()
        w = RI.dequantize_mxfp4(q).double()
        half = 0.0 if dtype == torch.float32 else torch.finfo(dtype).eps / 2
        for lo in range(0, N, 1 << 16):
            part = w[lo:lo + (1 << 16)].t()
            want, mass = a @ part, a.abs() @ part.abs()
            err = (out[:, lo:lo + (1 << 16)].double() - want).abs()
            assert (err <= H * 2.0 ** -23 * mass * (1 + half) + half * want.abs()).all(), lo


def test_linear_places(device):
    """Whole numbers that name their row, column and place in the row: nothing is exchanged, scales included."""
    M, N, H = 37, 150, 384
    for k in (0, 1, 31, 32, 63, 64, 95, 96, 127, 128, 200, 383):
        x, w = torch.zeros(M, H), torch.zeros(N, H)
        x[:, k] = torch.ldexp(torch.tensor([1.0, 1.5, 2.0, 3.0]).repeat(10)[:M], torch.arange(M) % 11 - 5)
        w[:, k] = torch.ldexp(torch.tensor([1.0, 1.5, 3.0, 4.0, -6.0]).repeat(30), torch.arange(N) % 17 - 8)
        got = RI.mxfp4_linear(x.to(device), RI.quantize_mxfp4(w.to(device)))
        assert torch.equal(got.cpu(), x[:, k, None] * w[None, :, k]), k


def test_linear_shapes_and_strides(device):
    g = torch.Generator().manual_seed(7)
    q = RI.quantize_mxfp4(torch.randn(70, 200, generator=g).to(device))
    x = torch.randn(3, 5, 433, generator=g).to(torch.bfloat16).to(device)
    for v in (x[..., 1:201], x[:, ::2, 8:208], x[0, 0, 3:203], x.transpose(0, 1)[..., :200], x[:1, :1, :200].expand(4, 9, 200),
              x[:0, :, :200]):
        out = RI.mxfp4_linear(v, q)
        assert out.shape == (*v.shape[:-1], 70)
        _check_linear(out, v, q)
    none = RI.MxFp4(q.codes[:0], q.scales[:0], 200)
    assert RI.mxfp4_linear(x[..., :200], none).shape == (3, 5, 0)


def test_linear_nan_blocks_and_extremes(device):
    """A block that is NaN makes its products NaN and no others; the largest and smallest blocks' products."""
    g = torch.Generator().manual_seed(11)
    x = torch.randn(20, 160, generator=g)
    w = torch.randn(50, 160, generator=g)
    x[3, 40] = math.nan
    w[7, 159] = math.inf
    x[5] = 0.0
    w[9, :64] = 0.0
    q = RI.quantize_mxfp4(w.to(device))
    _check_linear(RI.mxfp4_linear(x.to(device), q), x, q)
    for a, b in ((2.0 ** 60, 2.0 ** 50), (2.0 ** -60, 2.0 ** -50), (2.0 ** 100, 2.0 ** -100), (2.0 ** -120, 2.0 ** 120)):
        x = torch.randn(20, 160, generator=g) * a
        q = RI.quantize_mxfp4((torch.randn(50, 160, generator=g) * b).to(device))
        _check_linear(RI.mxfp4_linear(x.to(device), q), x, q)


def test_linear_captured_and_on_a_stream(device):
    g = torch.Generator().manual_seed(13)
    w = torch.randn(3000, 512, generator=g).to(torch.bfloat16).to(device)
    x = torch.randn(24, 512, generator=g).to(torch.bfloat16).to(device)
    RI.mxfp4_linear(x, RI.quantize_mxfp4(w))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        q = RI.quantize_mxfp4(w)
        out = RI.mxfp4_linear(x, q)
    side = torch.cuda.Stream(device=device)
    for k in range(3):
        x.copy_(torch.randn(24, 512, generator=g).to(device))
        w.copy_(torch.randn(3000, 512, generator=g).to(device) * (k + 1))
        graph.replay()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            want = RI.mxfp4_linear(x, RI.quantize_mxfp4(w))
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        _check_linear(out, x, q)


def test_draft_head_to_verified_tokens(device):
    """A speculative step as a rollout runs it: 4-bit draft head, sampler, target head, verification."""
    g = torch.Generator().manual_seed(17)
    B, K, H, V = 6, 3, 256, 4001
    head = (torch.randn(V, H, generator=g) * 0.2).to(torch.bfloat16).to(device)
    hidden = torch.randn(B, K + 1, H, generator=g).to(torch.bfloat16).to(device)
    q = RI.quantize_mxfp4(head)
    draft = RI.mxfp4_linear(hidden[:, :K], q)
    tokens = RI.sample_next_token_batch(draft.reshape(B * K, V), 1.0, 0, 1.0, True, seed=5).token_ids.view(B, K)
    target = hidden @ head.t()
    u = torch.rand(B, K + 1, generator=g).to(device)
    out = RI.verify_draft_tokens(target, tokens, draft, u)
    lp = torch.log_softmax(target.double(), -1)
    for b in range(B):
        n = int(out.num_accepted[b])
        assert torch.equal(out.token_ids[b, :n], tokens[b, :n])
        assert (out.token_ids[b, :n + 1] >= 0).all() and (out.token_ids[b, n + 1:] == -1).all()
        want = lp[b, torch.arange(n + 1), out.token_ids[b, :n + 1]]
        assert (out.logprobs[b, :n + 1].double() - want).abs().max() <= 2 ** -24 * want.abs().max() + 1e-11
    # the 4-bit head is near enough that most drafts are accepted
    assert out.num_accepted.sum() > B * K // 3
