"""MI355X-native token-sampling path (drop-in for Forgeline's sampler).

Public API
----------
apply_sampling_filters, sample_from_logits, generate_tokens
    Reference-compatible functions (src/forgeline/models/generation/sampling.py).
sample_tokens, describe_rows, filtered_outputs, SamplerPlan
    Batched entry points with heterogeneous per-row parameters (SamplerPlan:
    prepared once, one launch per decode step, capturable in a graph).
BatchedSampler
    A decode group's sampling state on the device (inference/engine.py:114-139).
speculative_verify, SpecPlan, SpeculativeGenerator, MTPSpeculativeGenerator
    Speculative-decoding accept / resample and the generators over B sequences
    (models/generation/speculative.py).
lm_head_sample, LmHeadPlan
    lm_head and sampling in one call, without the [B, V] logits
    (models/transformer/model.py:190, :201).
token_logprobs_from_logits, entropy_from_logits, kl_full_distribution, row_stats
    Full-distribution log-prob / entropy / KL in one pass (models/policy.py,
    training/common/logprobs.py).
score_tokens, score_tokens_backward
    Log-probabilities of given tokens with entropy, rank and top alternatives, and
    the logits' gradient (models/policy.py, training/common/logprobs.py).
lm_head_logprobs, lm_head_logprobs_backward
    The same from hidden states and the lm_head weight, without the [N, V] logits.
layer_norm, layer_norm_backward
    The norm in front of the head, with its gradients.
SamplingParams
    Per-request parameters with the reference's validation (inference/requests.py).
"""

from .params import GenerationSettings, SamplingParams, SamplingParamsError
from .sampling import (SampleOutput, SamplerPlan, SamplingError, apply_sampling_filters, describe_rows,
                       filtered_outputs, generate_tokens, sample_from_logits, sample_tokens)
from .speculative import MTPSpeculativeGenerator, SpeculativeGenerator, SpecOutput, SpecPlan, speculative_verify
from .engine import BatchedSampler
from .logprobs import RowStats, entropy_from_logits, kl_full_distribution, row_stats, token_logprobs_from_logits
from .norm import layer_norm, layer_norm_backward
from .scores import TokenScores, score_tokens, score_tokens_backward
from .lmhead import LmHeadOutput, LmHeadPlan, lm_head_sample
from .headlp import HeadScores, lm_head_logprobs, lm_head_logprobs_backward

__all__ = [
    "apply_sampling_filters", "sample_from_logits", "generate_tokens",
    "sample_tokens", "describe_rows", "filtered_outputs", "SampleOutput", "SamplerPlan", "SamplingError",
    "speculative_verify", "SpeculativeGenerator", "MTPSpeculativeGenerator", "SpecOutput", "SpecPlan",
    "BatchedSampler", "row_stats", "RowStats", "token_logprobs_from_logits", "entropy_from_logits", "kl_full_distribution",
    "SamplingParams", "GenerationSettings", "SamplingParamsError",
    "score_tokens", "score_tokens_backward", "TokenScores", "layer_norm", "layer_norm_backward",
    "lm_head_logprobs", "lm_head_logprobs_backward", "HeadScores",
    "lm_head_sample", "LmHeadPlan", "LmHeadOutput",
]
