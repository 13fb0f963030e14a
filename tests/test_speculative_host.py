"""Draft verification's argument checks, which run before any tensor reaches a
device, and the C entry point's host-side validation."""

from __future__ import annotations

import pytest
import torch

from rosellm_amd import _native as nat
from rosellm_amd.roseinfer import verify_draft_tokens as verify


def test_verify_refusals():
    x, y = torch.zeros(2, 4, 9), torch.zeros(2, 3, 9)
    d, u = torch.zeros(2, 3, dtype=torch.long), torch.zeros(2, 4)
    with pytest.raises(ValueError, match="3D"):
        verify(x[0], d, y, u)
    with pytest.raises(TypeError, match="float32, bfloat16 or float16"):
        verify(x.double(), d, y, u)
    with pytest.raises(ValueError, match="one position"):
        verify(x[:, :0], d, y, u)
    with pytest.raises(ValueError, match="vocabulary"):
        verify(x[..., :0], d, y, u)
    with pytest.raises(ValueError, match="draft_tokens"):
        verify(x, d[:, :2], y, u)
    with pytest.raises(TypeError, match="draft_tokens"):
        verify(x, d.float(), y, u)
    with pytest.raises(ValueError, match="draft_logits"):
        verify(x, d, x, u)
    with pytest.raises(TypeError, match="dtype of target"):
        verify(x, d, y.half(), u)
    with pytest.raises(ValueError, match="uniforms must"):
        verify(x, d, y, u[:, :3])
    with pytest.raises(TypeError, match="uniforms"):
        verify(x, d, y, u.double())
    with pytest.raises(ValueError, match="uniforms are needed"):
        verify(x, d, y, None)
    for t in (float("nan"), float("inf")):
        with pytest.raises(ValueError, match="finite"):
            verify(x, d, y, u, t)
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        verify(x, d, y, u)
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        verify(x, d, None, None, 0.0)


def test_verify_entry_point_validation():
    if not nat.LIB_PATH.exists():
        pytest.skip("librosellm_amd.so is not built (run __graft_entry__.build())")
    lib = nat.load()

    def run(x=16, y=16, dt=nat.BF16, B=2, K=3, V=9, drafts=16, ddt=nat.I64, u=16, T=1.0, sample=1, tok=16,
            cnt=16, lp=16, ws=16):
        return lib.rrl_verify_drafts(x, y, dt, B, K, V, 36, 9, 27, 9, nat.RrlView(drafts, ddt, 3, 1), u, T,
                                     sample, tok, cnt, lp, ws, None)

    assert run(B=0) == 0
    assert run(dt=nat.F64) == -2 and b"logits" in lib.rrl_last_error()
    assert run(ddt=nat.I16) == -2 and b"draft tokens" in lib.rrl_last_error()
    assert run(B=-1) == -1 and run(K=-1) == -1 and b"negative" in lib.rrl_last_error()
    assert run(V=0) == -1 and b"vocabulary" in lib.rrl_last_error()
    assert run(B=1 << 20, K=100, V=200000) == -1 and b"too large" in lib.rrl_last_error()
    assert run(T=float("nan")) == -1 and run(T=float("inf")) == -1
    for k in ("x", "drafts", "u", "tok", "cnt", "lp", "ws"):
        assert run(**{k: None}) == -1 and b"null" in lib.rrl_last_error(), k
    for k, bad in (("x", 17), ("y", 17), ("u", 18), ("ws", 8), ("drafts", 12)):
        assert run(**{k: bad}) == -4 and b"aligned" in lib.rrl_last_error(), k
    size = lib.rrl_verify_drafts_workspace_bytes
    assert size(2, 3, 9000, 1) >= 2 * 7 * 3 * 16 and size(2, 3, 9000, 0) < size(2, 3, 9000, 1)
    assert size(1 << 20, 100, 200000, 1) == 0 and size(-1, 3, 9, 1) == 0
