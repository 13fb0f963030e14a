"""The argument checks of adapter_linear, which run before any tensor reaches a device,
and the C entry points' host-side validation."""

from __future__ import annotations

import pytest
import torch

from rosellm_amd import _native as nat
from rosellm_amd import roseinfer
from rosellm_amd.rosetrainer import adapter_linear


def test_refusals():
    x, down, up = torch.zeros(5, 8), torch.zeros(3, 2, 8), torch.zeros(3, 6, 2)
    ids, base = torch.zeros(5, dtype=torch.long), torch.zeros(5, 6)
    assert roseinfer.adapter_linear is adapter_linear
    with pytest.raises(TypeError, match="x must be float32"):
        adapter_linear(x.double(), down, up, ids)
    for d, u in ((down[0], up), (down, up[0]), (down[:2], up), (down[:, :1], up)):
        with pytest.raises(ValueError, match=r"\[A, r, H\] and \[A, O, r\]"):
            adapter_linear(x, d, u, ids)
    for d, u in ((torch.zeros(3, 129, 8), torch.zeros(3, 6, 129)), (down[:0], up[:0]), (down[:, :0], up[:, :, :0]),
                 (down, up[:, :0]), (torch.zeros(4097, 1, 8), torch.zeros(4097, 6, 1))):
        with pytest.raises(ValueError, match="4096 adapters of rank 1 to 128"):
            adapter_linear(x, d, u, ids)
    with pytest.raises(ValueError, match="x must have shape"):
        adapter_linear(x[:, :7], down, up, ids)
    with pytest.raises(TypeError, match="the dtype of x"):
        adapter_linear(x.bfloat16(), down, up, ids)
    with pytest.raises(ValueError, match="adapter_ids are needed"):
        adapter_linear(x, down, up)
    with pytest.raises(TypeError, match="adapter_ids must be"):
        adapter_linear(x, down, up, ids.to(torch.int16))
    with pytest.raises(ValueError, match="adapter_ids must have shape"):
        adapter_linear(x, down, up, ids[:4])
    with pytest.raises(ValueError, match="base must have shape"):
        adapter_linear(x, down, up, ids, base=base[:, :5])
    with pytest.raises(TypeError, match="base must have the dtype"):
        adapter_linear(x, down, up, ids, base=base.half())
    for bad in (torch.ones(2), torch.ones(3, dtype=torch.float64)):
        with pytest.raises(ValueError, match="scales must be float32"):
            adapter_linear(x, down, up, ids, scales=bad)
    with pytest.raises(ValueError, match="scales have no gradient"):
        adapter_linear(x, down, up, ids, scales=torch.ones(3, requires_grad=True))
    with pytest.raises(ValueError, match=r"dropout_p must be in \[0, 1\]"):
        adapter_linear(x, down, up, ids, dropout_p=1.5)
    with pytest.raises(TypeError, match="offset"):
        adapter_linear(x, down, up, ids, dropout_p=0.5, offset=torch.zeros(2))
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        adapter_linear(x, down, up, ids, base=base)


@pytest.fixture(scope="module")
def lib():
    if not nat.LIB_PATH.exists():
        pytest.skip("librosellm_amd.so is not built (run __graft_entry__.build())")
    return nat.load()


def test_padded_ranks(lib):
    assert [lib.rrl_adapter_rank_padded(r) for r in (0, 1, 16, 17, 32, 33, 64, 65, 128, 129)] == [
        0, 16, 16, 32, 32, 64, 64, 128, 128, 0]


def test_entry_point_validation(lib):
    def params(dt=nat.BF16, N=4, H=8, O=6, A=2, r=3, down=16, up=16, ids=16, idt=nat.I64, scales=None, drop=None):
        return nat.RrlAdapterParams(dt, N, H, O, A, r, down, 24, 8, up, 18, 3, ids, idt, scales, drop)

    def fwd(x=16, ld=8, base=None, bld=0, out=16, t=16, **kw):
        return lib.rrl_adapter_fwd(params(**kw), x, ld, base, bld, out, t, None)

    def bwd(x=16, ld=8, g=16, gld=6, t=16, dx=16, dd=16, du=16, ws=16, **kw):
        return lib.rrl_adapter_bwd(params(**kw), x, ld, g, gld, t, dx, dd, du, ws, None)

    assert fwd(N=0) == 0 and lib.rrl_adapter_fwd(None, 16, 8, None, 0, 16, 16, None) == -1
    assert lib.rrl_adapter_bwd(None, 16, 8, 16, 6, 16, 16, 16, 16, 16, None) == -1
    for call in (fwd, bwd):
        assert call(dt=nat.F64) == -2 and b"float32" in lib.rrl_last_error()
        for bad in (dict(N=-1), dict(H=0), dict(O=0), dict(A=0), dict(r=0), dict(r=129), dict(A=4097),
                    dict(N=(1 << 30) + 1), dict(H=(1 << 24) + 1), dict(A=4096, r=128, H=1 << 20)):
            assert call(**bad) == -1 and b"bad size" in lib.rrl_last_error(), bad
        assert call(ids=None) == -1 and b"ids are needed" in lib.rrl_last_error()
        assert call(idt=nat.F32) == -2 and call(ids=12) == -4 and call(scales=2) == -4
        assert call(down=None) == -1 and call(up=None) == -1 and b"null" in lib.rrl_last_error()
        assert call(down=17) == -4 and call(up=17) == -4 and call(x=17) == -4
        assert call(ld=-1) == -1 and b"stride" in lib.rrl_last_error()
        import ctypes

        drop = nat.RrlDropoutParams(2.0, 0, 0, None)
        assert call(drop=ctypes.pointer(drop)) == -1 and b"probability" in lib.rrl_last_error()
    assert fwd(x=None) == -1 and fwd(out=None) == -1 and fwd(t=None) == -1 and fwd(out=17) == -4 and fwd(t=24) == -4
    assert fwd(base=17) == -4 and fwd(base=16, bld=-1) == -1
    assert bwd(g=None) == -1 and bwd(x=None) == -1 and bwd(t=None) == -1 and bwd(ws=None) == -1
    assert bwd(g=17) == -4 and bwd(dx=17) == -4 and bwd(dd=17) == -4 and bwd(du=17) == -4
    assert bwd(t=24) == -4 and bwd(ws=24) == -4 and bwd(gld=-1) == -1
    size = lib.rrl_adapter_bwd_workspace_bytes
    assert size(4, 8, 6, 2, 129, nat.BF16) == 0 and size(-1, 8, 6, 2, 3, nat.BF16) == 0
    # both factors turned, s, and a run's sums of both gradients
    assert size(1000, 64, 48, 2, 16, nat.BF16) >= 2 * 2 * 16 * 112 + 4 * 1000 * 16 + 4 * 2 * 16 * 112
