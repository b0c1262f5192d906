"""Scores of given tokens on MI355X, with gradients: the log-probability of each
row's token, the entropy, the token's rank and the top alternatives, from one
read of the logits.

``score_tokens`` serves a decode step's rows (one work-group per 16384 values,
so that few rows spread over the chip) and a training batch's alike.  Where
``logits`` requires a gradient, ``logprob``, ``entropy`` and ``lse`` carry one
(one more read of the logits and a write of their gradient); ``rank`` and the
alternatives do not.  The formulas are those of the reference's
``token_logprobs`` (``models/policy.py:47-50``) and ``entropy_from_logits``
(``training/common/logprobs.py:65-68``), except that a masked logit (-inf) adds
0 to the entropy, where the reference's ``0 * -inf`` is NaN.
"""

from __future__ import annotations

from dataclasses import dataclass
from typing import Optional

import torch

from . import _lib
from .logprobs import IGNORE_INDEX
from .sampling import _DTYPES

_INTS = (torch.int64, torch.int32, torch.int16, torch.int8, torch.uint8)


@dataclass
class TokenScores:
    logprob: Optional[torch.Tensor]        # float32 [...]
    entropy: Optional[torch.Tensor]        # float32 [...]
    lse: Optional[torch.Tensor]            # float32 [...]
    rank: Optional[torch.Tensor]           # int32 [...]: values greater than the token's (-1: no token)
    top_ids: Optional[torch.Tensor]        # int64 [..., top_k]
    top_logprobs: Optional[torch.Tensor]   # float32 [..., top_k]


def _check_logits(logits: torch.Tensor) -> None:
    if not isinstance(logits, torch.Tensor):
        raise TypeError("logits must be a torch.Tensor")
    if logits.device.type != "cuda":
        raise ValueError("logits must be on a ROCm device (no CPU fallback)")
    if logits.dtype not in _DTYPES:
        raise NotImplementedError(f"logits dtype {logits.dtype} is not supported (float32, bfloat16, float16)")
    if logits.dim() < 1 or logits.size(-1) < 1:
        raise ValueError("logits must have a vocabulary dimension of at least 1")


def _tokens(tokens: torch.Tensor, lead, dev: torch.device) -> torch.Tensor:
    if not isinstance(tokens, torch.Tensor) or tokens.dtype not in _INTS:
        raise TypeError("tokens must be a torch.Tensor of integers")
    if tokens.shape != lead:
        raise ValueError(f"tokens {tuple(tokens.shape)} must be {tuple(lead)}")
    if tokens.dtype != torch.int64 or tokens.device != dev or not tokens.is_contiguous():
        tokens = tokens.to(device=dev, dtype=torch.int64).contiguous()
    return tokens


def _no_autograd_under_capture(what: str, keep: str = "return_saved") -> None:
    """A backward pass recorded into a graph synchronises with the streams that
    other graphs of the same leaves ran on, which capture forbids and which can
    end the process: a captured step calls the functional form instead."""
    if torch.cuda.is_current_stream_capturing():
        raise RuntimeError(f"{what} does not record its autograd graph under stream capture: "
                           f"call it under torch.no_grad() with {keep}=True, then {what}_backward")


def _check_range(tokens: torch.Tensor, vocab: int, ignore_index: int) -> None:
    bad = ((tokens < 0) | (tokens >= vocab)) & (tokens != ignore_index)
    if bool(bad.any()):
        raise IndexError(f"token {int(tokens[bad][0])} is out of bounds for {vocab} classes")


def score_tokens(logits: torch.Tensor, tokens: Optional[torch.Tensor] = None, *, top_k: int = 0,
                 entropy: bool = False, lse: bool = False, rank: bool = False, ignore_index: int = IGNORE_INDEX,
                 check_tokens: bool = False, return_saved: bool = False):
    """Scores of ``logits [..., V]`` (float32, bfloat16 or float16): the
    log-probability of ``tokens [...]`` and its rank (``rank=True``: how many
    values are greater), the entropy, log-sum-exp, and the ``top_k`` (0 to 64)
    largest values' ids and log-probabilities, equal values by ascending id.

    A position whose token is ``ignore_index`` has log-probability -0.0, no
    gradient from it, and rank -1.  A token outside ``[0, V)`` gives NaN and
    rank -1; ``check_tokens=True`` raises ``IndexError`` instead (and waits for
    the device, as ``row_stats`` does).  A row with a NaN or +inf logit, or with
    -inf alone, has NaN results and ids -1; a -inf logit is a masked value, with
    probability and gradient 0.

    Differentiable (once, in reverse mode) in ``logits``, except under stream capture: a
    captured step takes ``return_saved=True``, which returns ``(scores, saved)``, under
    ``torch.no_grad()``, and ``score_tokens_backward``.  Nothing here waits for
    the device unless ``check_tokens`` is set."""
    _check_logits(logits)
    V = logits.size(-1)
    top_k = int(top_k)
    if not 0 <= top_k <= V:
        raise ValueError(f"top_k {top_k} must lie in 0 .. {V}")
    lead = logits.shape[:-1]
    tok = None
    if tokens is not None:
        tok = _tokens(tokens, lead, logits.device)
        if check_tokens:
            _check_range(tok, V, ignore_index)
    elif rank:
        raise ValueError("rank needs tokens")
    # (a call that asks for no result with a gradient has no graph)
    if logits.requires_grad and torch.is_grad_enabled() and (tok is not None or entropy or lse or return_saved):
        if return_saved:
            raise ValueError("return_saved is for calls under torch.no_grad()")
        _no_autograd_under_capture("score_tokens")
        out = iter(_lib.autograd().score(logits, tok, top_k, entropy, lse, rank, ignore_index))
        asked = (tok is not None, entropy, lse, rank, top_k, top_k)
        return TokenScores(*(next(out) if on else None for on in asked))
    out = _lib.autograd().score_forward(logits, tok, top_k, entropy, lse, rank, ignore_index, return_saved)
    s = TokenScores(*out[:6])
    return (s, out[6]) if return_saved else s


def _upstream(g: Optional[torch.Tensor], lead, dev: torch.device, name: str) -> Optional[torch.Tensor]:
    if g is None:
        return None
    if g.shape != lead or g.device != dev:
        raise ValueError(f"{name} must be {tuple(lead)} on {dev}")
    return g.to(torch.float32).contiguous()


def score_tokens_backward(logits: torch.Tensor, tokens: Optional[torch.Tensor], saved: torch.Tensor,
                          grad_logprob: Optional[torch.Tensor] = None, grad_entropy: Optional[torch.Tensor] = None,
                          grad_lse: Optional[torch.Tensor] = None, *, ignore_index: int = IGNORE_INDEX) -> torch.Tensor:
    """The gradient of ``sum(grad_logprob * logprob + grad_entropy * entropy +
    grad_lse * lse)`` with respect to ``logits``, in their dtype: what autograd
    computes for ``score_tokens``, as one launch that a graph may record.
    ``saved`` comes from ``score_tokens(..., return_saved=True)`` on the same
    logits and tokens (with ``entropy=True`` if ``grad_entropy`` is given)."""
    _check_logits(logits)
    dev, lead = logits.device, logits.shape[:-1]
    rows = logits.numel() // logits.size(-1)
    if saved.shape != (rows, 4) or saved.dtype != torch.float32 or saved.device != dev or not saved.is_contiguous():
        raise ValueError(f"saved must be the float32 [{rows}, 4] tensor of the forward call")
    tok = None if tokens is None else _tokens(tokens, lead, dev)
    if grad_logprob is not None and tok is None:
        raise ValueError("grad_logprob needs tokens")
    return _lib.autograd().score_backward(logits, tok, saved, _upstream(grad_logprob, lead, dev, "grad_logprob"),
                                          _upstream(grad_entropy, lead, dev, "grad_entropy"),
                                          _upstream(grad_lse, lead, dev, "grad_lse"), ignore_index)
