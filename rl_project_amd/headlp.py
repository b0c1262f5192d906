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

import ctypes
from dataclasses import dataclass
from functools import lru_cache
from typing import Optional, Tuple

import torch

from . import _lib
from ._lib import HeadArgs, HeadGradArgs, call, lib, ptr
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


def _hidden_rows(hidden: torch.Tensor) -> torch.Tensor:
    """[N, D] with rows that 16-byte loads can take (a copy where they cannot)."""
    h = hidden.reshape(-1, hidden.size(-1))
    if h.stride(1) != 1 or (h.size(0) > 1 and (h.stride(0) < h.size(1) or h.stride(0) % 8 or h.stride(0) > 1 << 21)):
        h = h.contiguous()
    if h.data_ptr() % 16:
        h = h.clone(memory_format=torch.contiguous_format)
    return h


@lru_cache(maxsize=256)
def _workspace_bytes(rows: int, vocab: int) -> int:
    n = ctypes.c_size_t(0)
    _lib.check(lib().fl_head_workspace_bytes(rows, vocab, ctypes.byref(n)), "fl_head_workspace_bytes")
    return n.value


@lru_cache(maxsize=256)
def _grad_workspace_bytes(rows: int, dim: int, vocab: int, dhidden: bool) -> int:
    n = ctypes.c_size_t(0)
    _lib.check(lib().fl_head_grad_workspace_bytes(rows, dim, vocab, int(dhidden), ctypes.byref(n)),
               "fl_head_grad_workspace_bytes")
    return n.value


def _forward(h, lead, weight, tok, entropy: bool, lse: bool, ignore_index: int, save: bool):
    R, D = h.shape
    V = weight.size(0)
    dev = h.device
    f32 = lambda shape: torch.empty(shape, dtype=torch.float32, device=dev)  # noqa: E731
    o_lp = f32(lead) if tok is not None else None
    o_h = f32(lead) if entropy else None
    o_lse = f32(lead) if lse else None
    saved = f32((R, 4)) if save else None
    n = _workspace_bytes(R, V) if D % 64 == 0 else 0
    ws = torch.empty(n, dtype=torch.uint8, device=dev)
    a = HeadArgs()
    a.struct_size = ctypes.sizeof(HeadArgs)
    a.dtype = _lib.FL_DTYPE_BF16
    a.hidden, a.weight = h.data_ptr(), weight.data_ptr()
    a.rows, a.dim, a.vocab, a.ld_hidden = R, D, V, h.stride(0) if R > 1 else D
    a.tokens, a.ignore_index = ptr(tok), ignore_index
    a.out_logprob, a.out_entropy, a.out_lse, a.out_saved = ptr(o_lp), ptr(o_h), ptr(o_lse), ptr(saved)
    a.workspace, a.workspace_bytes = ptr(ws), n
    call(lib().fl_head_logprobs, a, dev, "fl_head_logprobs")
    return o_lp, o_h, o_lse, saved


def _backward(h, shape, weight, tok, saved, ga, gb, gc, ignore_index: int, need_h: bool, need_w: bool):
    R, D = h.shape
    V = weight.size(0)
    dev = h.device
    dh = torch.empty(shape, dtype=torch.bfloat16, device=dev) if need_h else None
    # (no rows: no sums)
    dw = None if not need_w else (torch.zeros if R == 0 else torch.empty)(V, D, dtype=torch.bfloat16, device=dev)
    n = _grad_workspace_bytes(R, D, V, need_h)
    ws = torch.empty(n, dtype=torch.uint8, device=dev)
    a = HeadGradArgs()
    a.struct_size = ctypes.sizeof(HeadGradArgs)
    a.dtype = _lib.FL_DTYPE_BF16
    a.hidden, a.weight = h.data_ptr(), weight.data_ptr()
    a.rows, a.dim, a.vocab, a.ld_hidden = R, D, V, h.stride(0) if R > 1 else D
    a.tokens, a.ignore_index, a.saved = ptr(tok), ignore_index, saved.data_ptr()
    a.grad_logprob, a.grad_entropy, a.grad_lse = ptr(ga), ptr(gb), ptr(gc)
    a.out_dhidden, a.out_dweight = ptr(dh), ptr(dw)
    a.workspace, a.workspace_bytes = ptr(ws), n
    call(lib().fl_head_logprobs_grad, a, dev, "fl_head_logprobs_grad")
    return dh, dw


def lm_head_logprobs(hidden: torch.Tensor, weight: torch.Tensor, tokens: Optional[torch.Tensor] = None, *,
                     entropy: bool = False, lse: bool = False, norm=None, ignore_index: int = IGNORE_INDEX,
                     check_tokens: bool = False, return_saved: bool = False):
    """``score_tokens`` of the logits ``hidden @ weight.T`` (log-probability of
    ``tokens [...]``, entropy, log-sum-exp), for ``hidden [..., D]`` and ``weight
    [V, D]`` in bfloat16, D a multiple of 64, without writing the logits.  The
    logits are float32 sums, not rounded to bfloat16 as ``linear``'s are.
    ``norm=(weight, bias, eps)`` applies ``layer_norm`` to the hidden states
    first (the model's final norm).  Ignored and out-of-range tokens as in
    ``score_tokens``; up to 131072 rows.

    Differentiable in ``hidden`` and ``weight`` (and through ``norm``), except
    under stream capture: a captured step takes ``return_saved=True``, which
    returns ``(scores, saved)``, under ``torch.no_grad()``, and
    ``lm_head_logprobs_backward``.  The backward pass holds the logits' gradient
    of a chunk of the vocabulary in bfloat16 (512 MiB, or 32 KiB a row)."""
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
    if grad and (hidden.requires_grad or weight.requires_grad):
        if return_saved:
            raise ValueError("return_saved is for calls under torch.no_grad()")
        _no_autograd_under_capture("lm_head_logprobs")
        if tok is None and not entropy and not lse:
            raise ValueError("nothing is asked for: give tokens, entropy=True or lse=True")
        out = iter(_lib.autograd().head(hidden, weight, tok, bool(entropy), bool(lse), int(ignore_index)))
        return HeadScores(*(next(out) if on else None for on in (tok is not None, entropy, lse)))
    out = _forward(_hidden_rows(hidden), lead, weight, tok, entropy, lse, int(ignore_index), return_saved)
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
    with torch.no_grad():
        _check(hidden, weight)
        lead, dev = hidden.shape[:-1], hidden.device
        h = _hidden_rows(hidden)
        if saved.shape != (h.size(0), 4) or saved.dtype != torch.float32 or saved.device != dev or not saved.is_contiguous():
            raise ValueError(f"saved must be the float32 [{h.size(0)}, 4] tensor of the forward call")
        tok = None if tokens is None else _tokens(tokens, lead, dev)
        ga = _upstream(grad_logprob, lead, dev, "grad_logprob")
        gb = _upstream(grad_entropy, lead, dev, "grad_entropy")
        gc = _upstream(grad_lse, lead, dev, "grad_lse")
        if ga is not None and tok is None:
            raise ValueError("grad_logprob needs tokens")
        if not need_dhidden and not need_dweight:
            return None, None
        return _backward(h, hidden.shape, weight, tok, saved, ga, gb, gc, int(ignore_index), need_dhidden, need_dweight)
