"""Dropout whose mask is drawn again where it is needed instead of being stored.

The reference's models drop out after the embedding, the attention and the MLP with
``nn.Dropout`` (rosetrainer/model.py), which keeps a mask of a byte an entry for the
backward.  Here an entry's fate is a function of its place, a seed and an offset
(Philox4x32-10), so the backward draws it again, and the residual that the result is
added to is read in the same pass (``rrl_dropout``).
"""

from __future__ import annotations

from typing import Optional, Union

import torch
from torch import Tensor
from torch.autograd.function import once_differentiable

from .. import _native as nat
from .._graph import recorded
from .._random import dropout_arguments, dropout_params

__all__ = ["dropout"]


def _rows(x: Tensor):
    """x [..., H] as rows at one stride: (tensor, rows, H, stride)."""

    y = x.reshape(1) if x.dim() == 0 else x
    H = y.shape[-1]
    R = y.numel() // H if H else 0
    y = y.reshape(R, H)
    if H > 1 and y.stride(1) != 1:
        y = y.contiguous()
    return y, R, H, (y.stride(0) if R > 1 else H)


def _drop(x: Tensor, residual: Optional[Tensor], draw) -> Tensor:
    p, seed, offset, at = draw
    dev = nat.require_device(x, residual, at)
    rows, R, H, ld = _rows(x)
    res, _, _, r_ld = (None, 0, 0, 0) if residual is None else _rows(residual)
    out = torch.empty(x.shape, dtype=x.dtype, device=dev)
    nat.call_on(dev, "rrl_dropout", rows.data_ptr(), nat.dtype_code(x.dtype), R, H, ld, nat.ptr(res), r_ld,
                dropout_params(p, seed, offset, at), out.data_ptr(), nat.stream_ptr(dev))
    return out


class _Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x: Tensor, residual: Optional[Tensor], p: float, seed: int, offset: int, at: Optional[Tensor]):
        # saved, so that an offset that was changed before the backward raises there
        ctx.save_for_backward(at)
        ctx.args = (p, seed, offset)
        return _drop(x, residual, (p, seed, offset, at))

    @staticmethod
    @once_differentiable
    def backward(ctx, g: Tensor):
        (at,) = ctx.saved_tensors
        dx = _drop(g, None, (*ctx.args, at)) if ctx.needs_input_grad[0] else None
        return dx, (g if ctx.needs_input_grad[1] else None), None, None, None, None


def dropout(x: Tensor, p: float, *, seed: Optional[int] = None, offset: Union[int, Tensor] = 0,
            generator: Optional[torch.Generator] = None, residual: Optional[Tensor] = None) -> Tensor:
    """``x / (1 - p)`` where an entry is kept, 0 elsewhere (also for a NaN or an
    infinity), plus ``residual`` (of x's shape and dtype) if there is one: [..., H] in
    x's dtype (float32, bfloat16 or float16), summed in float32 and rounded once.

    An entry is dropped with probability ``p`` in [0, 1], to the nearest multiple of
    2^-16, by which the kept ones are scaled, so that the expectation is x's.  Its fate
    depends on its place, ``seed`` and ``offset`` alone: equal arguments give equal masks,
    whatever the strides, and the gradient draws the forward's mask again.  Give each
    call of a step a seed or an offset of its own, and a seed that
    ``sample_next_token_batch``, which draws from the same generator, does not have.
    With ``seed=None`` a seed is drawn from ``generator`` (a CPU ``torch.Generator``,
    default: torch's global one), on the host: a captured graph replays it, and a trace
    keeps it.  For another mask at each replay, ``offset`` can be an int64 tensor of one
    element on x's device, which the kernel reads; it must stay as it was until the
    backward has run (changing it in place before raises there).

    The mask is drawn in groups of eight entries along the last dimension, which are
    numbered through all rows; ``adapter_linear`` drops its input with the same one.  The
    call does not wait for the device; the gradient is not differentiable again.
    """

    if x.dtype not in (torch.float32, torch.bfloat16, torch.float16):
        raise TypeError("x must be float32, bfloat16 or float16")
    if residual is not None:
        if residual.shape != x.shape:
            raise ValueError(f"residual must have shape {tuple(x.shape)}, got {tuple(residual.shape)}")
        if residual.dtype != x.dtype:
            raise TypeError("residual must have the dtype of x")
    draw = dropout_arguments(p, seed, offset, generator, "p")
    if not recorded(x, residual):
        return _drop(x, residual, draw)
    return _Dropout.apply(x, residual, *draw)
