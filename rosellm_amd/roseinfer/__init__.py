"""MI355X-native pieces of ``rosellm.roseinfer`` on the RoseRLHF path: the
next-token sampler of roseinfer/engine.py:1088-1171, returning the behaviour
log-probabilities that rollout records need (roserlhf/trajectory.py:15,27-28);
the verification of drafted tokens, which returns them too; and a draft model's
head in microscaled 4-bit floating point."""

from .mxfp4 import MxFp4, dequantize_mxfp4, mxfp4_linear, quantize_mxfp4
from .sampling import SampleOutput, sample_next_token, sample_next_token_batch
from .speculative import VerifyOutput, verify_draft_tokens

__all__ = [
    "MxFp4",
    "SampleOutput",
    "VerifyOutput",
    "dequantize_mxfp4",
    "mxfp4_linear",
    "quantize_mxfp4",
    "sample_next_token",
    "sample_next_token_batch",
    "verify_draft_tokens",
]
