"""The token embedding with scaling, and its gradient by sorted tokens.

The reference's models look their input tokens up with ``nn.Embedding``
(rosetrainer/model.py, rosetrainer/qwen3.py), whose weight is the LM head's when
the two are tied.  Here the lookup and its scale are one pass, and the gradient
is formed from the positions sorted by token: every row of d weight is written
once, with no float atomics, so equal inputs give equal bits
(``rrl_embedding_fwd``, ``rrl_embedding_bwd``).
"""

from __future__ import annotations

import ctypes
import math
from typing import Optional

import torch
from torch import Tensor
from torch.autograd.function import once_differentiable

from .. import _native as nat

__all__ = ["embedding"]


class _Embedding(torch.autograd.Function):
    @staticmethod
    def forward(ctx, ids: Tensor, weight: Tensor, scale: float, padding_idx: Optional[int]):
        dev = nat.require_device(ids, weight)
        V, H = weight.shape
        w = weight if weight.stride(1) == 1 or H == 1 else weight.contiguous()
        w_ld = w.stride(0) if V > 1 else H
        if w_ld < H:  # rows that overlap or repeat (an expanded weight)
            w, w_ld = w.contiguous(), H
        flat = ids.reshape(-1).contiguous()
        out = torch.empty(*ids.shape, H, dtype=weight.dtype, device=dev)
        pad = (0, 0) if padding_idx is None else (padding_idx, 1)
        nat.call_on(dev, "rrl_embedding_fwd", flat.data_ptr(), nat.dtype_code(flat.dtype),
                    flat.numel(), w.data_ptr(), nat.dtype_code(w.dtype), V, H, w_ld, scale, *pad,
                    out.data_ptr(), nat.stream_ptr(dev))
        ctx.save_for_backward(ids)
        ctx.args = (V, H, weight.dtype, scale, pad)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, g: Tensor):
        (ids,) = ctx.saved_tensors
        V, H, dtype, scale, pad = ctx.args
        dev = g.device
        flat = ids.reshape(-1).contiguous()
        N = flat.numel()
        rows = g.reshape(N, H)
        if rows.stride(1) != 1 or (N > 1 and rows.stride(0) < H):  # as after an expand
            rows = rows.contiguous()
        dw = torch.empty(V, H, dtype=dtype, device=dev)
        ws = torch.empty(nat.lib().rrl_embedding_bwd_workspace_bytes(N, V, H), dtype=torch.uint8,
                         device=dev)
        nat.call_on(dev, "rrl_embedding_bwd", flat.data_ptr(), nat.dtype_code(flat.dtype), N,
                    rows.data_ptr(), nat.dtype_code(dtype), V, H, rows.stride(0) if N > 1 else H,
                    scale, *pad, dw.data_ptr(), H, ws.data_ptr(), nat.stream_ptr(dev))
        return None, dw, None, None


def embedding(token_ids: Tensor, weight: Tensor, *, scale: float = 1.0,
              padding_idx: Optional[int] = None) -> Tensor:
    """``scale * weight[token_ids]``: [..., H] in the weight's dtype for
    ``token_ids`` [...] (int32 or int64) and ``weight`` [V, H] (float32, bfloat16
    or float16).  The scale is taken as a float32 number (a finite one past
    float32's range is refused); the products are float32's, rounded to the
    weight's dtype.

    A token equal to ``padding_idx``, which may be negative (the -1 that
    ``roseinfer.verify_draft_tokens`` leaves past the last verified token), takes
    a row of zeros and passes no gradient.  The call does not wait for the device,
    so any other id outside ``[0, V)`` cannot raise: its row is NaN, and it passes
    no gradient.

    The gradient of ``weight`` is dense, in its dtype: float32 sums, in an order
    that the ids alone decide, times the scale, rounded once to the dtype.  It is
    not differentiable again.
    """

    if token_ids.dtype not in (torch.int64, torch.int32):
        raise TypeError("token_ids must be an int64 or int32 tensor")
    if weight.dim() != 2:
        raise ValueError(f"weight must be 2D [V, H], got shape={tuple(weight.shape)}")
    if weight.dtype not in (torch.float32, torch.bfloat16, torch.float16):
        raise TypeError("weight must be float32, bfloat16 or float16")
    if padding_idx is not None:
        padding_idx = int(padding_idx)
        if not -2 ** 63 <= padding_idx < 2 ** 63:
            raise ValueError("padding_idx must fit an int64")
    scale = float(scale)
    if math.isinf(ctypes.c_float(scale).value) and not math.isinf(scale):
        raise ValueError(f"scale {scale} is past float32's range")
    return _Embedding.apply(token_ids, weight, scale, padding_idx)
