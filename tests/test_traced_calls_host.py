"""What torch.jit.trace makes of calls that write their results through the native library."""

from __future__ import annotations

import pytest
import torch

from rosellm_amd._graph import recorded
from rosellm_amd.roseinfer import sample_tokens


def test_traced_calls_are_recorded():
    """A trace sees a call only as an autograd function: without one it would keep the empty result alone."""
    seen = []

    def f(x):
        seen.append(recorded(x))
        return x + 1

    torch.jit.trace(f, torch.ones(3), check_trace=False)
    assert seen == [True]
    assert not recorded(torch.ones(3))


def test_sampling_refuses_to_be_traced():
    with pytest.raises(RuntimeError, match="traced"):
        torch.jit.trace(lambda x: sample_tokens(x, torch.zeros(2))[0], torch.zeros(2, 5), check_trace=False)
