"""Low-rank adapters of many requests beside a shared projection, with gradients.

A policy that is trained as a low-rank adapter adds ``up (down x)`` to a projection of
the shared model.  In a rollout every request may be another policy's, so one batch
holds many adapters' rows; in training the input is dropped out, and both factors and
the input have gradients.  The reference's projections are ``F.linear``
(rosetrainer/model.py); it has no adapters.  The shared product itself is the
caller's (``F.linear``, ``roseinfer.mxfp4_linear``), and its result is the ``base`` that
is added in the same pass (``rrl_adapter_fwd``, ``rrl_adapter_bwd``).
"""

from __future__ import annotations

import ctypes
from typing import Optional, Union

import torch
from torch import Tensor
from torch.autograd.function import once_differentiable

from .. import _native as nat
from .._graph import recorded
from .._random import dropout_arguments, dropout_params

__all__ = ["adapter_linear"]

_MOST_ADAPTERS, _MOST_RANK = 4096, 128


def _rows(x: Tensor):
    """x [..., H] as rows at one stride: (tensor, stride)."""

    H = x.shape[-1]
    y = x.reshape(-1, H)
    if H > 1 and y.stride(1) != 1:
        y = y.contiguous()
    return y, (y.stride(0) if y.shape[0] > 1 else H)


def _factor(w: Tensor) -> Tensor:
    return w if w.stride(2) == 1 or w.shape[2] == 1 else w.contiguous()


def _params(dtype, N, down, up, ids, scales, drop):
    A, r, H = down.shape
    return nat.RrlAdapterParams(
        nat.dtype_code(dtype), N, H, up.shape[1], A, r, down.data_ptr(), down.stride(0), down.stride(1),
        up.data_ptr(), up.stride(0), up.stride(1), nat.ptr(ids), nat.dtype_code(ids.dtype) if ids is not None else 0,
        nat.ptr(scales), ctypes.pointer(drop) if drop is not None else None)


def _adapt(x, down, up, base, ids, scales, at, draw):
    """The result, and the rows' ``down x``."""

    dev = nat.require_device(x, down, up, base, ids, scales, at)
    rows, ld = _rows(x)
    N = rows.shape[0]
    flat = None if ids is None else ids.reshape(-1).contiguous()
    scales = None if scales is None else scales.contiguous()
    down, up = _factor(down), _factor(up)
    b, b_ld = (None, 0) if base is None else _rows(base)
    out = torch.empty(*x.shape[:-1], up.shape[1], dtype=x.dtype, device=dev)
    t = torch.empty(N, nat.lib().rrl_adapter_rank_padded(down.shape[1]), dtype=torch.float32, device=dev)
    drop = dropout_params(*draw, at) if draw is not None else None
    nat.call_on(dev, "rrl_adapter_fwd", _params(x.dtype, N, down, up, flat, scales, drop), rows.data_ptr(), ld,
                nat.ptr(b), b_ld, out.data_ptr(), t.data_ptr(), nat.stream_ptr(dev))
    return out, t


class _Adapter(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, down, up, base, ids, scales, at, draw):
        out, t = _adapt(x, down, up, base, ids, scales, at, draw)
        ctx.save_for_backward(x if ctx.needs_input_grad[1] else None, down, up, ids, scales,
                              t if ctx.needs_input_grad[2] else None, at)
        ctx.args = (x.shape, draw)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        x, down, up, ids, scales, t, at = ctx.saved_tensors
        shape, draw = ctx.args
        need_x, need_down, need_up, need_base = ctx.needs_input_grad[:4]
        dx = ddown = dup = None
        if need_x or need_down or need_up:
            dev = g.device
            down, up = _factor(down), _factor(up)
            scales = None if scales is None else scales.contiguous()
            rows, ld = _rows(g)
            N = rows.shape[0]
            A, r, H = down.shape
            xr, x_ld = (None, 0) if x is None else _rows(x)
            flat = None if ids is None else ids.reshape(-1).contiguous()
            if need_x:
                dx = torch.empty(shape, dtype=g.dtype, device=dev)
            if need_down:
                ddown = torch.empty(down.shape, dtype=g.dtype, device=dev)
            if need_up:
                dup = torch.empty(up.shape, dtype=g.dtype, device=dev)
            ws = torch.empty(nat.lib().rrl_adapter_bwd_workspace_bytes(N, H, up.shape[1], A, r, nat.dtype_code(g.dtype)),
                             dtype=torch.uint8, device=dev)
            drop = dropout_params(*draw, at) if draw is not None else None
            nat.call_on(dev, "rrl_adapter_bwd", _params(g.dtype, N, down, up, flat, scales, drop), nat.ptr(xr), x_ld,
                        rows.data_ptr(), ld, nat.ptr(t), nat.ptr(dx), nat.ptr(ddown), nat.ptr(dup), ws.data_ptr(),
                        nat.stream_ptr(dev))
        return dx, ddown, dup, (g if need_base else None), None, None, None, None


def adapter_linear(x: Tensor, down: Tensor, up: Tensor, adapter_ids: Optional[Tensor] = None, *,
                   base: Optional[Tensor] = None, scales: Optional[Tensor] = None, dropout_p: float = 0.0,
                   seed: Optional[int] = None, offset: Union[int, Tensor] = 0,
                   generator: Optional[torch.Generator] = None) -> Tensor:
    """``base + scales[a] * up[a] @ (down[a] @ x)`` for every row of ``x`` [..., H] with
    its own ``a = adapter_ids`` [...] (int32 or int64): [..., O] in x's dtype (float32,
    bfloat16 or float16).

    ``down`` [A, r, H] and ``up`` [A, O, r] hold A adapters of rank r (at most 4096 of
    rank 128; lower ranks are padded with zeros), ``base`` [..., O] the shared projection
    (``None``: zeros), all of x's dtype, and ``scales`` [A] float32 numbers without a
    gradient (``None``: ones).  A negative id is a row without an adapter, its result
    ``base`` alone; ``adapter_ids=None`` stands for the only adapter of A = 1.  The call
    does not wait for the device, so an id of A or more cannot raise: its row is NaN, and
    passes no gradient but to ``base``.

    ``dropout_p``, ``seed``, ``offset`` and ``generator`` are ``dropout``'s: x is dropped
    out within the product, as ``dropout(x, dropout_p, ...)`` of the same arguments would.
    Products are summed in float32, ``down[a] @ x`` is float32 between the two, and the
    result is rounded once.  x, ``down``, ``up`` and ``base`` have gradients, the factors'
    over all their rows in float32, in an order that the ids and sizes alone decide; they
    are not differentiable again.  An infinity among the operands stays in the sums that
    it enters, but as a NaN where a product was formed in parts.
    """

    if x.dtype not in (torch.float32, torch.bfloat16, torch.float16):
        raise TypeError("x must be float32, bfloat16 or float16")
    if down.dim() != 3 or up.dim() != 3 or down.shape[0] != up.shape[0] or down.shape[1] != up.shape[2]:
        raise ValueError(f"down and up must have shapes [A, r, H] and [A, O, r], got {tuple(down.shape)} "
                         f"and {tuple(up.shape)}")
    A, r, H = down.shape
    O = up.shape[1]
    if not 1 <= A <= _MOST_ADAPTERS or not 1 <= r <= _MOST_RANK or H < 1 or O < 1:
        raise ValueError(f"1 to {_MOST_ADAPTERS} adapters of rank 1 to {_MOST_RANK} are possible, got "
                         f"{tuple(down.shape)} and {tuple(up.shape)}")
    if x.dim() < 1 or x.shape[-1] != H:
        raise ValueError(f"x must have shape [..., {H}], got {tuple(x.shape)}")
    if down.dtype != x.dtype or up.dtype != x.dtype:
        raise TypeError("down and up must have the dtype of x")
    if adapter_ids is None:
        if A != 1:
            raise ValueError(f"adapter_ids are needed with {A} adapters")
    else:
        if adapter_ids.dtype not in (torch.int64, torch.int32):
            raise TypeError("adapter_ids must be an int64 or int32 tensor")
        if adapter_ids.shape != x.shape[:-1]:
            raise ValueError(f"adapter_ids must have shape {tuple(x.shape[:-1])}, got {tuple(adapter_ids.shape)}")
    if base is not None:
        if base.shape != (*x.shape[:-1], O):
            raise ValueError(f"base must have shape {(*x.shape[:-1], O)}, got {tuple(base.shape)}")
        if base.dtype != x.dtype:
            raise TypeError("base must have the dtype of x")
    if scales is not None:
        if tuple(scales.shape) != (A,) or scales.dtype != torch.float32:
            raise ValueError(f"scales must be float32 of shape {(A,)}")
        if scales.requires_grad:
            raise ValueError("scales have no gradient: detach them")
    dropout_p = float(dropout_p)
    draw = at = None
    if dropout_p != 0.0:
        *draw, at = dropout_arguments(dropout_p, seed, offset, generator, "dropout_p")
    if not recorded(x, down, up, base):
        return _adapt(x, down, up, base, adapter_ids, scales, at, draw)[0]
    return _Adapter.apply(x, down, up, base, adapter_ids, scales, at, draw)
