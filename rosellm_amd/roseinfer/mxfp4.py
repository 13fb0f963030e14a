"""Microscaled 4-bit floating point for a draft model's LM head.

Speculative rollouts verify every draft against the target's own distribution
(``verify_draft_tokens``), so the draft model's logits can be cheap ones: its
head kept in 4 bits takes 17/32 of a byte per weight and runs on the scaled
matrix instructions.  ``quantize_mxfp4`` lays a weight out once per policy
update, ``mxfp4_linear`` is ``x @ weight.T`` with ``x`` quantised the same way,
and its logits go to ``sample_next_token_batch`` and ``verify_draft_tokens``.
The reference's heads are ``F.linear`` in the weight's dtype
(rosetrainer/model.py:641); it has no quantised form.

The format is OCP MX: blocks of 32 entries along a row, e2m1 elements
(0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives) and a power-of-two scale,
``2^(floor(log2 max) - 2)``, held as a biased exponent byte; elements are
rounded to nearest, ties to even, and saturate at 6.
"""

from __future__ import annotations

from typing import NamedTuple, Optional

import torch
from torch import Tensor

from .. import _native as nat

__all__ = ["MxFp4", "dequantize_mxfp4", "mxfp4_linear", "quantize_mxfp4"]

_FLOATS = (torch.float32, torch.bfloat16, torch.float16)


class MxFp4(NamedTuple):
    """A matrix [R, cols] in blocks; with P = cols rounded up to a multiple of 128
    (the entries past cols are zeros)."""

    codes: Tensor   # [R, P / 2] uint8: two entries a byte, the first in the low four bits
    scales: Tensor  # [R, P / 32] uint8: exponent + 127; 255 marks a block that held NaN or infinity
    cols: int


def _padded(cols: int) -> int:
    return (cols + 127) // 128 * 128


def _rows(x: Tensor):
    """x [..., H] as rows at one stride: (tensor, rows, stride)."""

    H = x.shape[-1]
    R = x.numel() // H if H else 0
    y = x.reshape(R, H)
    if H > 1 and y.stride(1) != 1:
        y = y.contiguous()
    return y, R, (y.stride(0) if R > 1 else H)


def _check(q: MxFp4) -> None:
    codes, scales, cols = q
    if codes.dtype != torch.uint8 or scales.dtype != torch.uint8:
        raise TypeError("codes and scales must be uint8")
    if codes.dim() != 2 or scales.dim() != 2:
        raise ValueError("codes and scales must be 2D")
    P = _padded(cols)
    if cols < 1 or codes.shape[1] * 2 != P or tuple(scales.shape) != (codes.shape[0], P // 32):
        raise ValueError(f"codes {tuple(codes.shape)} and scales {tuple(scales.shape)} do not hold "
                         f"rows of {cols} entries")
    if not (codes.is_contiguous() and scales.is_contiguous()) or codes.data_ptr() % 16:
        raise ValueError("codes and scales must be contiguous, codes at a multiple of 16 bytes")


def quantize_mxfp4(x: Tensor) -> MxFp4:
    """``x`` [R, H] (float32, bfloat16 or float16) in microscaled 4-bit blocks
    along its rows.  A block with a NaN or an infinity stands for NaN."""

    if x.dim() != 2:
        raise ValueError(f"x must be 2D [R, H], got shape={tuple(x.shape)}")
    if x.dtype not in _FLOATS:
        raise TypeError("x must be float32, bfloat16 or float16")
    R, H = x.shape
    if H == 0:
        raise ValueError("x needs at least one column")
    dev = nat.require_device(x)
    rows, _, ld = _rows(x)
    P = _padded(H)
    codes = torch.empty(R, P // 2, dtype=torch.uint8, device=dev)
    scales = torch.empty(R, P // 32, dtype=torch.uint8, device=dev)
    nat.call_on(dev, "rrl_mxfp4_quantize", rows.data_ptr(), nat.dtype_code(x.dtype), R, H, ld,
                codes.data_ptr(), scales.data_ptr(), nat.stream_ptr(dev))
    return MxFp4(codes, scales, H)


def dequantize_mxfp4(q: MxFp4, dtype: torch.dtype = torch.float32) -> Tensor:
    """The numbers that the blocks stand for, [R, cols] (float32 and bfloat16 hold
    every one exactly, unless they are subnormal there)."""

    _check(q)
    if dtype not in _FLOATS:
        raise TypeError("dtype must be float32, bfloat16 or float16")
    dev = nat.require_device(q.codes, q.scales)
    R = q.codes.shape[0]
    out = torch.empty(R, q.cols, dtype=dtype, device=dev)
    nat.call_on(dev, "rrl_mxfp4_dequantize", q.codes.data_ptr(), q.scales.data_ptr(), R, q.cols,
                out.data_ptr(), nat.dtype_code(dtype), nat.stream_ptr(dev))
    return out


def mxfp4_linear(x: Tensor, weight: MxFp4, out_dtype: Optional[torch.dtype] = None) -> Tensor:
    """``x @ weight.T``: [..., R] for ``x`` [..., cols] (float32, bfloat16 or
    float16) and a weight of R rows from ``quantize_mxfp4``.

    ``x`` is quantised to the same blocks within the call; the products of the
    4-bit numbers are summed in float32 and rounded once to ``out_dtype``
    (default: x's).  There is no gradient: a draft head is not trained through
    its quantised form.
    """

    _check(weight)
    if x.dtype not in _FLOATS:
        raise TypeError("x must be float32, bfloat16 or float16")
    if x.dim() < 1 or x.shape[-1] != weight.cols:
        raise ValueError(f"x must have shape [..., {weight.cols}], got {tuple(x.shape)}")
    out_dtype = x.dtype if out_dtype is None else out_dtype
    if out_dtype not in _FLOATS:
        raise TypeError("out_dtype must be float32, bfloat16 or float16")
    dev = nat.require_device(x, weight.codes, weight.scales)
    rows, M, ld = _rows(x.detach())
    H, N = weight.cols, weight.codes.shape[0]
    # the kernel reads four scales at a time: a view at another address is moved
    scales = weight.scales if weight.scales.data_ptr() % 4 == 0 else weight.scales.clone()
    out = torch.empty(*x.shape[:-1], N, dtype=out_dtype, device=dev)
    ws = torch.empty(nat.lib().rrl_mxfp4_linear_workspace_bytes(M, H), dtype=torch.uint8, device=dev)
    nat.call_on(dev, "rrl_mxfp4_linear", rows.data_ptr(), nat.dtype_code(x.dtype), M, H, ld,
                weight.codes.data_ptr(), scales.data_ptr(), N, out.data_ptr(),
                nat.dtype_code(out_dtype), ws.data_ptr(), nat.stream_ptr(dev))
    return out
