"""Seeds and counters of the framework's counter-based random numbers."""

from __future__ import annotations

from typing import Optional, Tuple, Union

import torch
from torch import Tensor

from . import _native as nat

__all__ = ["dropout_arguments", "dropout_params", "draw_seed"]


def draw_seed(generator: Optional[torch.Generator]) -> int:
    """A 63-bit seed from a host generator (no device sync)."""

    return int(torch.randint(0, 2 ** 63 - 1, (1,), generator=generator, dtype=torch.int64).item())


def dropout_arguments(p: float, seed: Optional[int], offset: Union[int, Tensor],
                      generator: Optional[torch.Generator], name: str) -> Tuple[float, int, int, Optional[Tensor]]:
    """``p`` (the argument ``name``) and ``seed`` checked, and ``offset`` as a number and
    a tensor that is added to it on the device."""

    p = float(p)
    if not 0.0 <= p <= 1.0:
        raise ValueError(f"{name} must be in [0, 1], got {p}")
    at = None
    if isinstance(offset, Tensor):
        if offset.dtype != torch.int64 or offset.numel() != 1:
            raise TypeError("offset must be a number or an int64 tensor of one element")
        at, offset = offset, 0
    if seed is None:
        seed = draw_seed(generator)
    return p, int(seed) & (2 ** 64 - 1), int(offset) & (2 ** 64 - 1), at


def dropout_params(p: float, seed: int, offset: int, at: Optional[Tensor]) -> nat.RrlDropoutParams:
    return nat.RrlDropoutParams(p, seed, offset, nat.ptr(at))
