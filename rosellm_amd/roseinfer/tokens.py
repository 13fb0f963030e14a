"""Next tokens from given uniforms, with settings of their own for every row.

``sample_next_token_batch`` keeps the reference's rules: one temperature, top-k and
top-p for the whole batch, and a floor of 1e-9 under every candidate's probability.
``sample_tokens`` is for batches of requests that each bring their settings, min-p
among them, and for rollouts that have to be drawn from the distribution whose
log-probs they record: it has no floor, its uniforms are an argument (as
``verify_draft_tokens``'s are), and its borders are decided in 64-bit sums
(``rrl_sample_tokens``).
"""

from __future__ import annotations

import math
from typing import Union

import torch
from torch import Tensor

from .. import _native as nat
from .sampling import SampleOutput

__all__ = ["sample_tokens"]


def sample_tokens(
    logits: Tensor,
    uniforms: Tensor,
    *,
    temperature: Union[float, Tensor] = 1.0,
    top_k: Union[int, Tensor] = 0,
    top_p: Union[float, Tensor] = 1.0,
    min_p: Union[float, Tensor] = 0.0,
    sampling_logprobs: bool = True,
) -> SampleOutput:
    """One token per row of ``logits`` [B, V] (float32, bfloat16 or float16), drawn with
    ``uniforms`` [B] (float32 in [0, 1), such as ``torch.rand``'s).

    A setting is one number, or a tensor of B numbers (float32; ``top_k``: int32 or
    int64) on the logits' device.  With ``p = softmax(logits / temperature)`` a row keeps

    * the ``top_k`` largest entries (off at 0 or less, and from V on), ties lowest index
      first;
    * of these, in descending order, those up to which their share of the sum of these is
      at most ``top_p`` (off outside (0, 1)), the first always;
    * of these, those of at least ``min_p`` times the largest probability (off at 0 or
      less; above 1 it counts as 1);

    and the token is the first, in vocabulary order, at which the running sum of what is
    kept exceeds the row's uniform times its whole (a uniform of 1 takes the last that has
    any).  A temperature of 0 or less takes the first maximum, whatever the other settings.

    The sums that decide this count a probability in units of 2^-44 of the largest one, to
    the nearest (of 2^-42 for the longest rows, V is at most 2^20): all of them together are
    off by at most V 2^-45 of it, 2^-27 for 2^18 entries and 2^-23 for 2^20, where a step
    of the uniforms is 2^-24; a product below one unit counts as 0.  Log-probs come from
    float64 sums.

    Returns the tokens, their ``log_softmax(logits / temperature)`` (at temperature 1
    where it is greedy) and, unless ``sampling_logprobs=False``, the log-probs of the
    distribution that was drawn from (0 where greedy).  The call does not wait for the
    device, so a row that has no distribution (a NaN or +inf among its logits or as its
    temperature, or nothing above -inf) cannot raise: its token is -1 and its log-probs
    are NaN.  It cannot be traced by ``torch.jit.trace``; a graph captures it.
    """

    if logits.dim() != 2:
        raise ValueError(f"logits must be 2D [B, V], got shape={tuple(logits.shape)}")
    if logits.dtype not in (torch.float32, torch.bfloat16, torch.float16):
        raise TypeError("logits must be float32, bfloat16 or float16")
    B, V = logits.shape
    if V == 0:
        raise ValueError("logits need at least one vocabulary entry")
    if tuple(uniforms.shape) != (B,):
        raise ValueError(f"uniforms must have shape {(B,)}, got {tuple(uniforms.shape)}")
    if uniforms.dtype != torch.float32:
        raise TypeError("uniforms must be float32")
    rows = {}
    for name, value, dtypes in (("temperature", temperature, (torch.float32,)),
                                ("top_k", top_k, (torch.int32, torch.int64)),
                                ("top_p", top_p, (torch.float32,)),
                                ("min_p", min_p, (torch.float32,))):
        if not isinstance(value, Tensor):
            if name != "top_k" and not math.isfinite(value):
                raise ValueError(f"{name} must be finite")
            continue
        if tuple(value.shape) != (B,):
            raise ValueError(f"{name} must be a number or have shape {(B,)}, got {tuple(value.shape)}")
        if value.dtype not in dtypes:
            raise TypeError(f"{name} must be " + " or ".join(str(d)[6:] for d in dtypes))
        rows[name] = value
    if torch.jit.is_tracing():
        raise RuntimeError("sample_tokens cannot be traced: a trace would not hold the kernels that write its results")
    dev = nat.require_device(logits, uniforms, *rows.values())

    x = logits if logits.stride(1) == 1 or V == 1 else logits.contiguous()
    u = uniforms.contiguous()
    rows = {name: value.contiguous() for name, value in rows.items()}
    params = nat.RrlSampleParams(
        *(0.0 if name in rows else float(value)
          for name, value in (("temperature", temperature), ("top_p", top_p), ("min_p", min_p))),
        0 if "top_k" in rows else max(0, min(int(top_k), V)),
        *(nat.ptr(rows.get(name)) for name in ("temperature", "top_p", "min_p", "top_k")),
        nat.dtype_code(rows["top_k"].dtype) if "top_k" in rows else 0)
    tokens = torch.empty(B, dtype=torch.int64, device=dev)
    logp = torch.empty(B, dtype=torch.float32, device=dev)
    logq = torch.empty(B, dtype=torch.float32, device=dev) if sampling_logprobs else None
    ws = torch.empty(nat.lib().rrl_sample_tokens_workspace_bytes(B, V, params), dtype=torch.uint8, device=dev)
    nat.call_on(dev, "rrl_sample_tokens", x.data_ptr(), nat.dtype_code(x.dtype), B, V,
                x.stride(0) if B > 1 else V, u.data_ptr(), params, tokens.data_ptr(), logp.data_ptr(),
                nat.ptr(logq), ws.data_ptr(), nat.stream_ptr(dev))
    return SampleOutput(tokens, logp, logq)
