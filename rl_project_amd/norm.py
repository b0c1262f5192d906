"""Layer norm on MI355X, forward and backward, as the norm in front of the head
uses it (``lm_head_sample`` and ``lm_head_logprobs`` take one as ``norm=``)."""

from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import _lib
from .sampling import _DTYPES
from .scores import _no_autograd_under_capture


def _check_x(x: torch.Tensor, name: str) -> None:
    if not isinstance(x, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if x.device.type != "cuda":
        raise ValueError(f"{name} must be on a ROCm device (no CPU fallback)")
    if x.dtype not in _DTYPES:
        raise NotImplementedError(f"{name} dtype {x.dtype} is not supported (float32, bfloat16, float16)")
    if x.dim() < 1 or x.size(-1) < 1:
        raise ValueError(f"{name} must have a last dimension of at least 1")


def _check_affine(x: torch.Tensor, weight: Optional[torch.Tensor], bias: Optional[torch.Tensor]) -> None:
    for t, name in ((weight, "weight"), (bias, "bias")):
        if t is None:
            continue
        if t.dim() != 1 or t.size(0) != x.size(-1) or t.device != x.device:
            raise ValueError(f"{name} must be [{x.size(-1)}] on {x.device}")
        if t.dtype != x.dtype and t.dtype != torch.float32:
            raise NotImplementedError(f"{name} dtype {t.dtype} is neither x's nor float32")
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise NotImplementedError("weight and bias must share a dtype")


def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
               eps: float = 1e-5, *, return_stats: bool = False):
    """``(x - mean) / sqrt(var + eps) * weight + bias`` over the last dimension of
    ``x [..., D]`` (float32, bfloat16 or float16; D up to 16384), in ``x``'s
    dtype; mean and variance (over D, not D - 1) in float32.  ``weight`` and
    ``bias`` (``[D]``, either may be None) share one dtype, ``x``'s or float32.

    Differentiable (once, in reverse mode) in all three, except under stream
    capture: a captured step takes ``return_stats=True``, which returns ``(y, stats)``, under
    ``torch.no_grad()``, and ``layer_norm_backward``."""
    _check_x(x, "x")
    _check_affine(x, weight, bias)
    if torch.is_grad_enabled() and (x.requires_grad or (weight is not None and weight.requires_grad)
                                    or (bias is not None and bias.requires_grad)):
        if return_stats:
            raise ValueError("return_stats is for calls under torch.no_grad()")
        _no_autograd_under_capture("layer_norm", "return_stats")
        return _lib.autograd().layer_norm(x, weight, bias, eps)
    y, stats = _lib.autograd().norm_forward(x, weight, bias, eps, return_stats)
    return (y, stats) if return_stats else y


def layer_norm_backward(grad: torch.Tensor, x: torch.Tensor, weight: Optional[torch.Tensor], bias: Optional[torch.Tensor],
                        stats: torch.Tensor, *, need_dx: bool = True, need_dweight: bool = True, need_dbias: bool = True
                        ) -> Tuple[Optional[torch.Tensor], Optional[torch.Tensor], Optional[torch.Tensor]]:
    """``(dx, dweight, dbias)`` of ``layer_norm`` for the upstream gradient
    ``grad``: what autograd computes, as launches that a graph may record.
    ``stats`` (float32 ``[2, rows]``: means, then reciprocal standard deviations)
    comes from ``layer_norm(..., return_stats=True)`` on the same ``x``.  The
    weight's and bias' gradients (None without a weight or bias, or where not
    needed) have their dtype; the sums over the rows have a fixed order."""
    _check_x(x, "x")
    _check_affine(x, weight, bias)
    if grad.shape != x.shape or grad.dtype != x.dtype or grad.device != x.device:
        raise ValueError("grad must match x in shape, dtype and device")
    rows = x.numel() // x.size(-1)
    if stats.shape != (2, rows) or stats.dtype != torch.float32 or stats.device != x.device or not stats.is_contiguous():
        raise ValueError(f"stats must be the forward call's float32 [2, {rows}] tensor")
    return tuple(_lib.autograd().norm_backward(grad, x, weight, bias, stats, need_dx, need_dweight, need_dbias))
