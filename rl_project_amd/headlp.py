"""Log-probabilities of given tokens from hidden states and the lm_head weight, with
gradients, without the ``[N, V]`` logits: the training and evaluation
counterpart of ``lm_head_sample``.

The reference computes ``logits = lm_head(h)`` (``transformer/model.py:176-179``)
and takes ``token_logprobs`` (``models/policy.py:47-50``) and
``entropy_from_logits`` (``training/common/logprobs.py:65-68``) of them.  Here
the softmax's statistics are taken from the product's float32 accumulators, and
the backward pass computes the logits again, a chunk of the vocabulary at a time.
"""

from __future__ import annotations

from dataclasses import dataclass
from typing import Optional, Tuple

import torch

from . import _lib
from .lmhead import _normed
from .logprobs import IGNORE_INDEX
from .scores import _check_range, _no_autograd_under_capture, _tokens, _upstream


@dataclass
class HeadScores:
    logprob: Optional[torch.Tensor]   # float32 [...]
    entropy: Optional[torch.Tensor]   # float32 [...]
    lse: Optional[torch.Tensor]       # float32 [...]


def _check(hidden: torch.Tensor, weight: torch.Tensor) -> None:
    if not isinstance(hidden, torch.Tensor) or not isinstance(weight, torch.Tensor):
        raise TypeError("hidden and weight must be torch.Tensors")
    if hidden.dim() < 1 or weight.dim() != 2 or hidden.size(-1) != weight.size(1):
        raise ValueError(f"hidden [..., D] and weight [V, D] expected, got {tuple(hidden.shape)} and {tuple(weight.shape)}")
    if hidden.dtype != torch.bfloat16 or weight.dtype != torch.bfloat16:
        raise NotImplementedError("lm_head_logprobs takes bf16 hidden states and weights")
    if hidden.device.type != "cuda" or hidden.device != weight.device:
        raise ValueError("hidden and weight must be on the same ROCm device (no CPU fallback)")
    if not weight.is_contiguous():
        raise ValueError("weight must be contiguous")
    if weight.size(0) < 1 or weight.size(1) < 1:
        raise ValueError("weight must have a row and a column")


def lm_head_logprobs(hidden: torch.Tensor, weight: torch.Tensor, tokens: Optional[torch.Tensor] = None, *,
                     entropy: bool = False, lse: bool = False, norm=None, ignore_index: int = IGNORE_INDEX,
                     check_tokens: bool = False, return_saved: bool = False):
    """``score_tokens`` of the logits ``hidden @ weight.T`` (log-probability of
    ``tokens [...]``, entropy, log-sum-exp), for ``hidden [..., D]`` and ``weight
    [V, D]`` in bfloat16, D a multiple of 64, without writing the logits.  The
    logits are float32 sums, not rounded to bfloat16 as ``linear``'s are.
    ``norm=(weight, bias, eps)`` applies ``layer_norm`` to the hidden states
    first (the model's final norm).  Ignored and out-of-range tokens as in
    ``score_tokens``; up to 131072 rows.  (The gradient of ``weight`` is a product
    over all rows: a NaN in the hidden states of an ignored row is in it too.)

    Differentiable (once, in reverse mode) in ``hidden`` and ``weight`` (and through
    ``norm``), except under stream capture: a captured step takes
    ``return_saved=True``, which returns ``(scores, saved)``, under
    ``torch.no_grad()``, and ``lm_head_logprobs_backward``.

    The backward pass holds the logits' gradient g of a chunk of the vocabulary in
    bfloat16 (512 MiB, or 32 KiB a row).  An entry loses at most 2^-8 of itself, as
    every entry does that a linear layer in bfloat16 is handed, so ``hidden``'s
    gradient is off by at most 2^-8 of ``sum_v |g| |weight|`` and ``weight``'s by 2^-8
    of ``sum_n |g| |hidden|``; the loss at a row's own token, the largest entry of
    most rows, is made good.  Against the rounding of the results themselves: 1.00
    to 1.07 times as far from 64 bits in random batches of 4099 tokens or more, up to
    1.35 times with 64 to 512, up to 2.4 times for rows whose probability sits on
    another token.  Where that matters, ``score_tokens`` over float32 logits keeps g
    in float32."""
    _check(hidden, weight)
    lead = hidden.shape[:-1]
    tok = None
    if tokens is not None:
        tok = _tokens(tokens, lead, hidden.device)
        if check_tokens:
            _check_range(tok, weight.size(0), ignore_index)
    grad = torch.is_grad_enabled()
    if grad and norm is not None and return_saved and any(isinstance(t, torch.Tensor) and t.requires_grad for t in norm[:2]):
        raise ValueError("return_saved is for calls under torch.no_grad()")
    hidden = _normed(hidden, norm)
    # (a call that asks for no result has no graph)
    if grad and (hidden.requires_grad or weight.requires_grad) and (tok is not None or entropy or lse or return_saved):
        if return_saved:
            raise ValueError("return_saved is for calls under torch.no_grad()")
        _no_autograd_under_capture("lm_head_logprobs")
        out = iter(_lib.autograd().head(hidden, weight, tok, entropy, lse, ignore_index))
        return HeadScores(*(next(out) if on else None for on in (tok is not None, entropy, lse)))
    out = _lib.autograd().head_forward(hidden, weight, tok, entropy, lse, ignore_index, return_saved)
    s = HeadScores(*out[:3])
    return (s, out[3]) if return_saved else s


def lm_head_logprobs_backward(hidden: torch.Tensor, weight: torch.Tensor, tokens: Optional[torch.Tensor],
                              saved: torch.Tensor, grad_logprob: Optional[torch.Tensor] = None,
                              grad_entropy: Optional[torch.Tensor] = None, grad_lse: Optional[torch.Tensor] = None, *,
                              need_dhidden: bool = True, need_dweight: bool = True, ignore_index: int = IGNORE_INDEX
                              ) -> Tuple[Optional[torch.Tensor], Optional[torch.Tensor]]:
    """``(dhidden, dweight)`` of ``lm_head_logprobs`` (without a norm) for the
    upstream gradients: what autograd computes, as launches that a graph may
    record.  ``saved`` comes from ``lm_head_logprobs(..., return_saved=True)`` on
    the same tensors (with ``entropy=True`` if ``grad_entropy`` is given)."""
    _check(hidden, weight)
    lead, dev = hidden.shape[:-1], hidden.device
    rows = hidden.numel() // hidden.size(-1)
    if saved.shape != (rows, 4) or saved.dtype != torch.float32 or saved.device != dev or not saved.is_contiguous():
        raise ValueError(f"saved must be the float32 [{rows}, 4] tensor of the forward call")
    tok = None if tokens is None else _tokens(tokens, lead, dev)
    if grad_logprob is not None and tok is None:
        raise ValueError("grad_logprob needs tokens")
    return tuple(_lib.autograd().head_backward(hidden, weight, tok, saved, _upstream(grad_logprob, lead, dev, "grad_logprob"),
                                               _upstream(grad_entropy, lead, dev, "grad_entropy"),
                                               _upstream(grad_lse, lead, dev, "grad_lse"), ignore_index, need_dhidden,
                                               need_dweight))
