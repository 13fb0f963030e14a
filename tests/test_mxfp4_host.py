"""The 4-bit head's argument checks, which run before any tensor reaches a
device, and the C entry points' host-side validation."""

from __future__ import annotations

import pytest
import torch

from rosellm_amd import _native as nat
from rosellm_amd.roseinfer import MxFp4, dequantize_mxfp4, mxfp4_linear, quantize_mxfp4


def _q(R=5, cols=200, P=256):
    return MxFp4(torch.zeros(R, P // 2, dtype=torch.uint8), torch.zeros(R, P // 32, dtype=torch.uint8), cols)


def test_mxfp4_refusals():
    x = torch.zeros(3, 200)
    with pytest.raises(ValueError, match="2D"):
        quantize_mxfp4(x[0])
    with pytest.raises(TypeError, match="float32"):
        quantize_mxfp4(x.double())
    with pytest.raises(ValueError, match="column"):
        quantize_mxfp4(x[:, :0])
    with pytest.raises(ValueError, match="do not hold"):
        dequantize_mxfp4(_q(cols=300))
    with pytest.raises(ValueError, match="do not hold"):
        dequantize_mxfp4(_q()._replace(scales=torch.zeros(4, 8, dtype=torch.uint8)))
    with pytest.raises(ValueError, match="do not hold"):
        dequantize_mxfp4(_q(cols=0, P=0))
    with pytest.raises(ValueError, match="2D"):
        dequantize_mxfp4(_q()._replace(scales=torch.zeros(8, dtype=torch.uint8)))
    with pytest.raises(TypeError, match="uint8"):
        dequantize_mxfp4(_q()._replace(codes=torch.zeros(5, 128)))
    with pytest.raises(ValueError, match="contiguous"):
        dequantize_mxfp4(_q()._replace(codes=torch.zeros(128, 5, dtype=torch.uint8).t()))
    with pytest.raises(TypeError, match="dtype"):
        dequantize_mxfp4(_q(), torch.float64)
    with pytest.raises(ValueError, match="shape"):
        mxfp4_linear(x[:, :100], _q())
    with pytest.raises(TypeError, match="x must"):
        mxfp4_linear(x.double(), _q())
    with pytest.raises(TypeError, match="out_dtype"):
        mxfp4_linear(x, _q(), torch.int32)
    for call in (lambda: quantize_mxfp4(x), lambda: dequantize_mxfp4(_q()), lambda: mxfp4_linear(x, _q())):
        with pytest.raises(RuntimeError, match="ROCm GPU"):
            call()


def test_mxfp4_entry_point_validation():
    if not nat.LIB_PATH.exists():
        pytest.skip("librosellm_amd.so is not built (run __graft_entry__.build())")
    lib = nat.load()

    def quant(x=16, dt=nat.BF16, R=2, H=64, ld=64, c=16, s=16):
        return lib.rrl_mxfp4_quantize(x, dt, R, H, ld, c, s, None)

    def dequant(c=16, s=16, R=2, H=64, out=16, dt=nat.BF16):
        return lib.rrl_mxfp4_dequantize(c, s, R, H, out, dt, None)

    def linear(x=16, dt=nat.BF16, M=2, H=64, ld=64, c=16, s=16, N=3, out=16, odt=nat.F32, ws=16):
        return lib.rrl_mxfp4_linear(x, dt, M, H, ld, c, s, N, out, odt, ws, None)

    assert quant(R=0) == 0 and dequant(R=0) == 0 and linear(M=0) == 0 and linear(N=0) == 0
    for call in (quant, dequant, linear):
        assert call(dt=nat.F64) == -2 and call(H=-1) == -1 and call(c=None) == -1 and call(s=None) == -1
        assert call(c=8) == -4 and b"aligned" in lib.rrl_last_error()
        assert call(H=1 << 32) == -1 and b"2^30" in lib.rrl_last_error()
    assert quant(x=None) == -1 and quant(x=17) == -4 and quant(ld=-1) == -1 and quant(R=-1) == -1
    assert dequant(out=None) == -1 and dequant(out=17) == -4 and dequant(R=-1) == -1
    assert linear(x=None) == -1 and linear(out=None) == -1 and linear(ws=None) == -1 and linear(H=0) == -1
    assert linear(odt=nat.I8) == -2 and linear(out=18) == -4 and linear(ws=8) == -4 and linear(x=17) == -4
    assert linear(ld=-1) == -1
    assert lib.rrl_mxfp4_linear_workspace_bytes(3, 200) >= 3 * (128 + 8)
    assert lib.rrl_mxfp4_linear_workspace_bytes(-1, 200) == 0
