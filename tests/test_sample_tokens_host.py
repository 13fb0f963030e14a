"""The argument checks of sample_tokens, which run before any tensor reaches a device,
its oracle on rows worked out by hand, and the C entry point's host-side validation."""

from __future__ import annotations

import math

import pytest
import torch

from rosellm_amd import _native as nat
from rosellm_amd.roseinfer import sample_tokens

from _sample_oracle import choose


def test_refusals():
    x, u = torch.zeros(3, 8), torch.zeros(3)
    with pytest.raises(ValueError, match="2D"):
        sample_tokens(x[0], u)
    with pytest.raises(TypeError, match="logits must be float32"):
        sample_tokens(x.double(), u)
    with pytest.raises(ValueError, match="vocabulary"):
        sample_tokens(x[:, :0], u)
    with pytest.raises(ValueError, match="uniforms must have shape"):
        sample_tokens(x, u[:2])
    with pytest.raises(TypeError, match="uniforms must be float32"):
        sample_tokens(x, u.double())
    for name in ("temperature", "top_p", "min_p"):
        with pytest.raises(ValueError, match=f"{name} must be finite"):
            sample_tokens(x, u, **{name: math.nan})
        with pytest.raises(ValueError, match=f"{name} must be a number or have shape"):
            sample_tokens(x, u, **{name: torch.ones(2)})
        with pytest.raises(TypeError, match=f"{name} must be float32"):
            sample_tokens(x, u, **{name: torch.ones(3, dtype=torch.float64)})
    with pytest.raises(TypeError, match="top_k must be int32 or int64"):
        sample_tokens(x, u, top_k=torch.ones(3))
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        sample_tokens(x, u)


def test_oracle_by_hand():
    x = torch.log(torch.tensor([0.1, 0.4, 0.2, 0.3], dtype=torch.float64))
    at = lambda u, **kw: choose(x, u, kw.get("T", 1.0), kw.get("k", 0), kw.get("tp", 1.0), kw.get("mp", 0.0))
    assert [at(u)[0] for u in (0.0, 0.05, 0.2, 0.55, 0.8)] == [0, 0, 1, 2, 3]
    assert at(0.9, k=2) == (3, pytest.approx(math.log(0.3)), pytest.approx(math.log(0.3 / 0.7)))
    assert at(0.9, tp=0.69)[0] == 1 and at(0.9, tp=0.71)[0] == 3
    assert at(0.99, tp=0.1)[0] == 1  # the first always
    assert at(0.0, mp=0.6)[0] == 1 and at(0.99, mp=0.74)[0] == 3 and at(0.99, mp=0.76)[0] == 1
    # top_p of what top_k leaves: 4/7 and 3/7
    assert at(0.99, k=2, tp=0.6)[0] == 1 and at(0.99, k=3, tp=0.6)[0] == 1
    assert at(0.5, T=0.0) == (1, pytest.approx(math.log(0.4)), 0.0)
    assert choose(torch.zeros(4), 0.9, 1.0, 2, 1.0, 0.0)[0] == 1  # ties: lowest index first
    assert choose(torch.full((4,), -math.inf), 0.9, 1.0, 2, 1.0, 0.0)[0] == -1


@pytest.fixture(scope="module")
def lib():
    if not nat.LIB_PATH.exists():
        pytest.skip("librosellm_amd.so is not built (run __graft_entry__.build())")
    return nat.load()


def test_entry_point_validation(lib):
    def call(x=16, dt=nat.BF16, B=2, V=8, ld=8, u=16, T=None, tp=None, mp=None, k=None, kdt=nat.I32, tok=16, lp=16,
             ws=16, params=True):
        p = nat.RrlSampleParams(1.0, 1.0, 0.0, 0, T, tp, mp, k, kdt) if params else None
        return lib.rrl_sample_tokens(x, dt, B, V, ld, u, p, tok, lp, None, ws, None)

    assert call(B=0) == 0
    assert call(dt=nat.F64) == -2 and b"float32" in lib.rrl_last_error()
    assert call(B=-1) == -1 and b"negative" in lib.rrl_last_error()
    assert call(V=0) == -1 and b"vocabulary" in lib.rrl_last_error()
    assert call(B=1 << 22) == -1 and call(V=(1 << 30) + 1) == -1 and b"2^30" in lib.rrl_last_error()
    for missing in ("x", "u", "tok", "lp", "ws"):
        assert call(**{missing: None}) == -1 and b"null" in lib.rrl_last_error()
    assert call(params=False) == -1
    assert call(ld=-8) == -1
    assert call(k=16, kdt=nat.F32) == -2 and b"top_k" in lib.rrl_last_error()
    assert call(x=17) == -4 and call(u=18) == -4 and call(T=2) == -4 and call(tp=2) == -4 and call(mp=2) == -4
    assert call(ws=8) == -4 and call(k=2) == -4 and call(k=12, kdt=nat.I64) == -4 and b"aligned" in lib.rrl_last_error()
    size = lib.rrl_sample_tokens_workspace_bytes
    assert size(-1, 8, None) == 0 and size(1, 0, None) == 0 and size(1 << 22, 8, None) == 0
    none, both = nat.RrlSampleParams(1.0, 1.0, 0.0, 0), nat.RrlSampleParams(1.0, 0.9, 0.0, 5)
    # histograms of 1024 sums and counts a part of 4096 entries, where there may be a cut
    assert size(4, 8192, both) == size(4, 8192, None) >= 4 * 2 * 1024 * 12 > size(4, 8192, none) > 0
