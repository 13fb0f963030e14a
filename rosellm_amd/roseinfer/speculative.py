"""Verification of drafted tokens (speculative sampling) with behaviour log-probs.

A draft model proposes K tokens per sequence; one pass of the target model gives
its logits at those K places and one more.  ``verify_draft_tokens`` keeps the
longest run of drafts that speculative sampling accepts, draws one more token,
and returns, as ``sample_next_token_batch`` does, the behaviour log-probability
of every token that it leaves.  Where the drafts were drawn from the softmax of the
draft logits that it is given, the tokens are distributed as if the target had
sampled them one by one, so they are rollout tokens like any others
(``PolicyAction.old_logprobs``, roserlhf/trajectory.py:15,27-28).
``sample_next_token_batch`` draws from ``max(q, 1e-9)``, which lies up to V 1e-9 of
the mass from that (1.5e-4 at 151,936 entries), and so far at most may a token's
distribution then lie from the target's; the log-probs are the target's all the
same.  The reference decodes one token per step (roseinfer/engine.py:1103-1171) and
has no such step.
"""

from __future__ import annotations

import math
from typing import NamedTuple, Optional

import torch
from torch import Tensor

from .. import _native as nat

__all__ = ["VerifyOutput", "verify_draft_tokens"]


class VerifyOutput(NamedTuple):
    token_ids: Tensor     # [B, K + 1] int64: the accepted drafts, one token more, then -1
    num_accepted: Tensor  # [B] int64: how many drafts were accepted
    logprobs: Tensor      # [B, K + 1] float32: log_softmax(target / T)[token], 0 past the last


def verify_draft_tokens(
    target_logits: Tensor,
    draft_tokens: Tensor,
    draft_logits: Optional[Tensor],
    uniforms: Optional[Tensor],
    temperature: float = 1.0,
    *,
    do_sample: bool = True,
) -> VerifyOutput:
    """Verify ``draft_tokens`` [B, K] (int32 or int64) against ``target_logits``
    [B, K + 1, V] (float32, bfloat16 or float16).

    ``draft_logits`` [B, K, V], in the target's dtype, are the logits that the
    drafts were sampled from at the same ``temperature``; ``None`` stands for
    drafts that were chosen without chance (copied from the prompt).  With
    ``p = softmax(target / T)`` and ``q = softmax(draft / T)`` (1 at the draft
    without draft logits), draft j is accepted while ``uniforms[b, j] * q < p``
    at its token.  The next token is drawn with ``uniforms[b, K]`` by inverse CDF
    in vocabulary order, from ``max(p - q, 0)`` after a rejection, else from
    ``p``; also from ``p`` where the two rows are equal (to 2^-35 of ``p``, what
    rounding can make of equal ones) and the draft has no mass in either.
    ``uniforms`` [B, K + 1] are float32 in [0, 1), such as
    ``torch.rand``'s.  A negative draft token ends its sequence's draft, so that
    drafts of different lengths can be padded with -1; the logits behind its
    end are not looked at.

    Logits of -inf have no probability, so a filter (top-k, top-p, a grammar) can
    be applied to both sides' logits beforehand.  With ``do_sample=False`` or
    ``temperature <= 0`` a draft is accepted while it is the target's first
    maximum, ``draft_logits`` and ``uniforms`` are not looked at, and the
    log-probs are those at temperature 1.

    The call does not wait for the device, so rows that have no distribution (a
    NaN or +inf among the logits, or nothing above -inf) and drafts of V or more
    cannot raise: the sequence ends there, with token -1 and a NaN log-prob.
    Exponentials and sums are float64, so that a token does not depend on the
    order in which 150,000 probabilities were added.
    """

    if target_logits.dim() != 3:
        raise ValueError(f"target_logits must be 3D [B, K + 1, V], got shape={tuple(target_logits.shape)}")
    if target_logits.dtype not in (torch.float32, torch.bfloat16, torch.float16):
        raise TypeError("target_logits must be float32, bfloat16 or float16")
    B, K, V = target_logits.shape[0], target_logits.shape[1] - 1, target_logits.shape[2]
    if K < 0:
        raise ValueError("target_logits need at least one position")
    if V == 0:
        raise ValueError("target_logits need at least one vocabulary entry")
    if tuple(draft_tokens.shape) != (B, K):
        raise ValueError(f"draft_tokens must have shape {(B, K)}, got {tuple(draft_tokens.shape)}")
    if draft_tokens.dtype not in (torch.int64, torch.int32):
        raise TypeError("draft_tokens must be an int64 or int32 tensor")
    temperature = float(temperature)
    if not math.isfinite(temperature):
        raise ValueError("temperature must be finite")
    greedy = (not do_sample) or temperature <= 0.0
    if greedy:
        draft_logits = uniforms = None
    else:
        if uniforms is None:
            raise ValueError("uniforms are needed to sample")
        if tuple(uniforms.shape) != (B, K + 1):
            raise ValueError(f"uniforms must have shape {(B, K + 1)}, got {tuple(uniforms.shape)}")
        if uniforms.dtype != torch.float32:
            raise TypeError("uniforms must be float32")
    if draft_logits is not None:
        if tuple(draft_logits.shape) != (B, K, V):
            raise ValueError(f"draft_logits must have shape {(B, K, V)}, got {tuple(draft_logits.shape)}")
        if draft_logits.dtype != target_logits.dtype:
            raise TypeError("draft_logits must have the dtype of target_logits")
    dev = nat.require_device(target_logits, draft_tokens, draft_logits, uniforms)

    x = target_logits if target_logits.stride(2) == 1 else target_logits.contiguous()
    y = draft_logits
    if y is not None and y.stride(2) != 1:
        y = y.contiguous()
    u = None if uniforms is None else uniforms.contiguous()
    tokens = torch.empty(B, K + 1, dtype=torch.int64, device=dev)
    count = torch.empty(B, dtype=torch.int64, device=dev)
    logp = torch.empty(B, K + 1, dtype=torch.float32, device=dev)
    ws = torch.empty(nat.lib().rrl_verify_drafts_workspace_bytes(B, K, V, int(y is not None)),
                     dtype=torch.uint8, device=dev)
    drafts = nat.RrlView(draft_tokens.data_ptr(), nat.dtype_code(draft_tokens.dtype),
                         draft_tokens.stride(0), draft_tokens.stride(1))
    nat.call_on(dev, "rrl_verify_drafts", x.data_ptr(), nat.ptr(y), nat.dtype_code(x.dtype), B, K, V,
                x.stride(0), x.stride(1), y.stride(0) if y is not None else 0,
                y.stride(1) if y is not None else 0, drafts, nat.ptr(u), temperature, int(not greedy),
                tokens.data_ptr(), count.data_ptr(), logp.data_ptr(), ws.data_ptr(),
                nat.stream_ptr(dev))
    return VerifyOutput(tokens, count, logp)
