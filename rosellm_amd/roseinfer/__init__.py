"""MI355X-native pieces of ``rosellm.roseinfer`` on the RoseRLHF path: the
next-token sampler of roseinfer/engine.py:1088-1171, returning the behaviour
log-probabilities that rollout records need (roserlhf/trajectory.py:15,27-28);
tokens from given uniforms with settings of their own for every request; the
verification of drafted tokens, which returns them too; a draft model's
head in microscaled 4-bit floating point; and the low-rank adapters of many
requests beside a shared projection."""

from ..rosetrainer.adapters import adapter_linear
from .mxfp4 import MxFp4, dequantize_mxfp4, mxfp4_linear, quantize_mxfp4
from .sampling import SampleOutput, sample_next_token, sample_next_token_batch
from .speculative import VerifyOutput, verify_draft_tokens
from .tokens import sample_tokens

__all__ = [
    "MxFp4",
    "SampleOutput",
    "VerifyOutput",
    "adapter_linear",
    "dequantize_mxfp4",
    "mxfp4_linear",
    "quantize_mxfp4",
    "sample_next_token",
    "sample_next_token_batch",
    "sample_tokens",
    "verify_draft_tokens",
]
