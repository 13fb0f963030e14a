"""The token embedding's argument checks, which run before any tensor reaches a
device, and the C entry points' host-side validation."""

from __future__ import annotations

import pytest
import torch

from rosellm_amd import _native as nat
from rosellm_amd.rosetrainer import embedding


def test_embedding_refusals():
    ids, w = torch.zeros(3, dtype=torch.long), torch.zeros(4, 8)
    with pytest.raises(TypeError, match="token_ids"):
        embedding(ids.float(), w)
    with pytest.raises(TypeError, match="token_ids"):
        embedding(ids.to(torch.int16), w)
    with pytest.raises(ValueError, match="2D"):
        embedding(ids, torch.zeros(8))
    with pytest.raises(TypeError, match="float32, bfloat16 or float16"):
        embedding(ids, w.double())
    with pytest.raises(ValueError, match="int64"):
        embedding(ids, w, padding_idx=2 ** 63)
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        embedding(ids, w)


@pytest.fixture(scope="module")
def lib():
    if not nat.LIB_PATH.exists():
        pytest.skip("librosellm_amd.so is not built (run __graft_entry__.build())")
    return nat.load()


def test_embedding_entry_point_validation(lib):
    def fwd(ids=16, idt=nat.I64, N=2, w=16, dt=nat.BF16, V=4, H=8, ld=8, out=16):
        return lib.rrl_embedding_fwd(ids, idt, N, w, dt, V, H, ld, 1.0, 0, 0, out, None)

    def bwd(ids=16, idt=nat.I64, N=2, g=16, dt=nat.BF16, V=4, H=8, gld=8, dw=16, dwld=8, ws=16):
        return lib.rrl_embedding_bwd(ids, idt, N, g, dt, V, H, gld, 1.0, 0, 0, dw, dwld, ws, None)

    assert fwd(N=0) == 0 and fwd(H=0) == 0 and bwd(V=0) == 0 and bwd(H=0) == 0
    for call in (fwd, bwd):
        assert call(dt=nat.F64) == -2 and b"float32" in lib.rrl_last_error()
        assert call(idt=nat.F32) == -2 and b"int32 or int64" in lib.rrl_last_error()
        assert call(N=-1) == -1 and b"negative" in lib.rrl_last_error()
        assert call(N=1 << 28) == -1 and b"2^28" in lib.rrl_last_error()
        assert call(V=1 << 26) == -1 and b"2^26" in lib.rrl_last_error()
        assert call(ids=None) == -1 and b"null" in lib.rrl_last_error()
        assert call(ids=12) == -4 and b"aligned" in lib.rrl_last_error()
    assert fwd(w=None) == -1 and fwd(out=None) == -1 and fwd(ld=7) == -1
    assert fwd(w=17) == -4 and fwd(out=17) == -4
    assert bwd(g=None) == -1 and bwd(dw=None) == -1 and bwd(ws=None) == -1
    assert bwd(gld=7) == -1 and bwd(dwld=7) == -1
    assert bwd(g=17) == -4 and bwd(dw=17) == -4 and bwd(ws=8) == -4
    assert lib.rrl_embedding_bwd_workspace_bytes(-1, 1, 1) == 0
    # sorted keys and positions twice, two bounds per row, a float32 row per 64 positions
    assert lib.rrl_embedding_bwd_workspace_bytes(6400, 500, 32) >= 16 * 6400 + 8 * 500 + 4 * 100 * 32
