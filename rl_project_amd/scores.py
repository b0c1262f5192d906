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

import ctypes
from dataclasses import dataclass
from functools import lru_cache
from typing import Optional

import torch

from . import _lib
from ._lib import ScoreArgs, ScoreGradArgs, call, lib, ptr
from .logprobs import IGNORE_INDEX, _rows
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


def _logits(logits: torch.Tensor) -> torch.Tensor:
    if isinstance(logits, torch.Tensor) and logits.dim() and logits.size(-1) < 1:
        raise ValueError("logits must have a vocabulary of at least 1")
    return _rows(logits, "logits")


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


@lru_cache(maxsize=256)
def _workspace_bytes(rows: int, vocab: int, top_k: int) -> int:
    n = ctypes.c_size_t(0)
    _lib.check(lib().fl_score_workspace_bytes(rows, vocab, top_k, ctypes.byref(n)), "fl_score_workspace_bytes")
    return n.value


def _forward(x: torch.Tensor, lead, tok: Optional[torch.Tensor], top_k: int, entropy: bool, lse: bool, rank: bool,
             ignore_index: int, save: bool):
    """The launch; (logprob, entropy, lse, rank, top_ids, top_logprobs, saved)."""
    R, V = x.shape
    dev = x.device
    L = lib()
    f32 = lambda shape: torch.empty(shape, dtype=torch.float32, device=dev)  # noqa: E731
    o_lp = f32(lead) if tok is not None else None
    o_h = f32(lead) if entropy else None
    o_lse = f32(lead) if lse else None
    o_rank = torch.empty(lead, dtype=torch.int32, device=dev) if rank else None
    o_ids = torch.empty((*lead, top_k), dtype=torch.int64, device=dev) if top_k else None
    o_top = f32((*lead, top_k)) if top_k else None
    saved = f32((R, 4)) if save else None
    a = ScoreArgs()
    a.struct_size = ctypes.sizeof(ScoreArgs)
    a.dtype = _DTYPES[x.dtype]
    a.logits = x.data_ptr()
    a.rows, a.vocab, a.ld = R, V, x.stride(0) if R > 1 else V
    a.tokens, a.ignore_index, a.top_k = ptr(tok), ignore_index, top_k
    a.out_logprob, a.out_entropy, a.out_lse, a.out_rank = ptr(o_lp), ptr(o_h), ptr(o_lse), ptr(o_rank)
    a.out_top_ids, a.out_top_logprobs, a.out_saved = ptr(o_ids), ptr(o_top), ptr(saved)
    ws = None
    if V > 16384 and R > 0:   # (rows of one slice need none)
        n = _workspace_bytes(R, V, top_k)
        ws = torch.empty(n, dtype=torch.uint8, device=dev)
        a.workspace, a.workspace_bytes = ws.data_ptr(), n
    call(L.fl_score_tokens, a, dev, "fl_score_tokens")
    return o_lp, o_h, o_lse, o_rank, o_ids, o_top, saved


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

    Differentiable in ``logits``, except under stream capture: a captured step
    takes ``return_saved=True``, which returns ``(scores, saved)``, under
    ``torch.no_grad()``, and ``score_tokens_backward``.  Nothing here waits for
    the device unless ``check_tokens`` is set."""
    x = _logits(logits)
    V = x.size(1)
    top_k = int(top_k)
    if not 0 <= top_k <= V:
        raise ValueError(f"top_k {top_k} must lie in 0 .. {V}")
    lead = logits.shape[:-1]
    tok = None
    if tokens is not None:
        tok = _tokens(tokens, lead, x.device)
        if check_tokens:
            _check_range(tok, V, ignore_index)
    elif rank:
        raise ValueError("rank needs tokens")
    if logits.requires_grad and torch.is_grad_enabled():
        if return_saved:
            raise ValueError("return_saved is for calls under torch.no_grad()")
        _no_autograd_under_capture("score_tokens")
        if top_k > _lib.FL_SCORE_MAX_TOPK:
            raise NotImplementedError(f"top_k {top_k} beyond the library's limit {_lib.FL_SCORE_MAX_TOPK}")
        out = iter(_lib.autograd().score(logits, tok, top_k, bool(entropy), bool(lse), bool(rank), int(ignore_index)))
        asked = (tok is not None, entropy, lse, rank, top_k, top_k)
        return TokenScores(*(next(out) if on else None for on in asked))
    out = _forward(x, lead, tok, top_k, entropy, lse, rank, int(ignore_index), return_saved)
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
    with torch.no_grad():
        x = _logits(logits)
        R, V = x.shape
        dev, lead = x.device, logits.shape[:-1]
        if saved.shape != (R, 4) or saved.dtype != torch.float32 or saved.device != dev or not saved.is_contiguous():
            raise ValueError(f"saved must be the float32 [{R}, 4] tensor of the forward call")
        tok = None if tokens is None else _tokens(tokens, lead, dev)
        ga = _upstream(grad_logprob, lead, dev, "grad_logprob")
        gb = _upstream(grad_entropy, lead, dev, "grad_entropy")
        gc = _upstream(grad_lse, lead, dev, "grad_lse")
        if ga is not None and tok is None:
            raise ValueError("grad_logprob needs tokens")
        out = torch.empty(logits.shape, dtype=x.dtype, device=dev)
        a = ScoreGradArgs()
        a.struct_size = ctypes.sizeof(ScoreGradArgs)
        a.dtype = _DTYPES[x.dtype]
        a.logits = x.data_ptr()
        a.rows, a.vocab, a.ld = R, V, x.stride(0) if R > 1 else V
        a.tokens, a.ignore_index, a.saved = ptr(tok), int(ignore_index), saved.data_ptr()
        a.grad_logprob, a.grad_entropy, a.grad_lse = ptr(ga), ptr(gb), ptr(gc)
        a.out_grad, a.out_ld = out.data_ptr(), V
        call(lib().fl_score_tokens_grad, a, dev, "fl_score_tokens_grad")
        return out
