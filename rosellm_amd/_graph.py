"""Whether a call has to be recorded: for a gradient, or by a trace."""

from __future__ import annotations

from typing import Optional

import torch
from torch import Tensor
from torch.autograd import forward_ad

__all__ = ["recorded"]


def recorded(*tensors: Optional[Tensor]) -> bool:
    """Whether autograd has to see a call on these: ``Function.apply`` takes 3 us of the
    host even where nothing needs a gradient, a quarter of a decode step's call.  Within
    forward-mode differentiation it does see it, and raises.  ``torch.jit.trace`` knows a
    call by its function alone: without one it would keep the empty result, and not what
    the kernel writes into it."""

    if getattr(forward_ad, "_current_level", 0) >= 0 or torch.jit.is_tracing():
        return True
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)
