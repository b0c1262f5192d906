"""Layer norm on MI355X, forward and backward, as the norm in front of the head
uses it (``lm_head_sample`` and ``lm_head_logprobs`` take one as ``norm=``)."""

from __future__ import annotations

import ctypes
from functools import lru_cache
from typing import NamedTuple, Optional, Tuple

import torch

from . import _lib
from ._lib import NormArgs, NormGradArgs, call, lib, ptr
from .sampling import _DTYPES
from .scores import _no_autograd_under_capture


class NormStats(NamedTuple):
    mean: torch.Tensor   # float32 [rows]
    rstd: torch.Tensor   # float32 [rows]


def _x_rows(x: torch.Tensor, name: str) -> torch.Tensor:
    if not isinstance(x, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if x.device.type != "cuda":
        raise ValueError(f"{name} must be on a ROCm device (no CPU fallback)")
    if x.dtype not in _DTYPES:
        raise NotImplementedError(f"{name} dtype {x.dtype} is not supported (float32, bfloat16, float16)")
    if x.dim() < 1 or x.size(-1) < 1:
        raise ValueError(f"{name} must have a last dimension of at least 1")
    if x.dim() == 2 and x.is_contiguous():
        return x
    x2 = x.reshape(-1, x.size(-1))
    if (x2.size(1) > 1 and x2.stride(1) != 1) or (x2.size(0) > 1 and x2.stride(0) < x2.size(1)):
        x2 = x2.contiguous()
    return x2


def _affine(t: Optional[torch.Tensor], x: torch.Tensor, name: str) -> Optional[torch.Tensor]:
    if t is None:
        return None
    if t.shape != (x.size(-1),) or t.device != x.device:
        raise ValueError(f"{name} must be [{x.size(-1)}] on {x.device}")
    if t.dtype != x.dtype and t.dtype != torch.float32:
        raise NotImplementedError(f"{name} dtype {t.dtype} is neither x's nor float32")
    return t.contiguous()


def _wdtype(x, weight, bias) -> int:
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise NotImplementedError("weight and bias must share a dtype")
    t = weight if weight is not None else bias
    return _DTYPES[x.dtype if t is None else t.dtype]


def _forward(x2, lead_shape, weight, bias, eps: float, stats: bool):
    R, D = x2.shape
    dev = x2.device
    y = torch.empty(lead_shape, dtype=x2.dtype, device=dev)
    mean = rstd = None
    a = NormArgs()
    a.struct_size = ctypes.sizeof(NormArgs)
    a.dtype, a.wdtype, a.eps = _DTYPES[x2.dtype], _wdtype(x2, weight, bias), eps
    a.x, a.rows, a.dim, a.ld = x2.data_ptr(), R, D, x2.stride(0) if R > 1 else D
    a.weight, a.bias = ptr(weight), ptr(bias)
    a.out, a.out_ld = y.data_ptr(), D
    if stats:
        mean = torch.empty(R, dtype=torch.float32, device=dev)
        rstd = torch.empty(R, dtype=torch.float32, device=dev)
        a.out_mean, a.out_rstd = mean.data_ptr(), rstd.data_ptr()
    call(lib().fl_layer_norm, a, dev, "fl_layer_norm")
    return y, mean, rstd


def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
               eps: float = 1e-5, *, return_stats: bool = False):
    """``(x - mean) / sqrt(var + eps) * weight + bias`` over the last dimension of
    ``x [..., D]`` (float32, bfloat16 or float16; D up to 16384), in ``x``'s
    dtype; mean and variance (over D, not D - 1) in float32.  ``weight`` and
    ``bias`` (``[D]``, either may be None) share one dtype, ``x``'s or float32.

    Differentiable in all three, except under stream capture: a captured step
    takes ``return_stats=True``, which returns ``(y, stats)``, under
    ``torch.no_grad()``, and ``layer_norm_backward``."""
    x2 = _x_rows(x, "x")
    eps = float(eps)
    if torch.is_grad_enabled() and (x.requires_grad or (weight is not None and weight.requires_grad)
                                    or (bias is not None and bias.requires_grad)):
        if return_stats:
            raise ValueError("return_stats is for calls under torch.no_grad()")
        _no_autograd_under_capture("layer_norm", "return_stats")
        _wdtype(x, _affine(weight, x, "weight"), _affine(bias, x, "bias"))
        return _lib.autograd().layer_norm(x, weight, bias, eps)
    y, mean, rstd = _forward(x2, x.shape, _affine(weight, x, "weight"), _affine(bias, x, "bias"), eps, return_stats)
    return (y, NormStats(mean, rstd)) if return_stats else y


def layer_norm_backward(grad: torch.Tensor, x: torch.Tensor, weight: Optional[torch.Tensor], bias: Optional[torch.Tensor],
                        stats: NormStats, *, need_dx: bool = True, need_dweight: bool = True, need_dbias: bool = True
                        ) -> Tuple[Optional[torch.Tensor], Optional[torch.Tensor], Optional[torch.Tensor]]:
    """``(dx, dweight, dbias)`` of ``layer_norm`` for the upstream gradient
    ``grad``: what autograd computes, as launches that a graph may record.
    ``stats`` comes from ``layer_norm(..., return_stats=True)`` on the same
    ``x``.  The weight's and bias' gradients (None without a weight or bias, or
    where not needed) have their dtype; the sums over the rows have a fixed
    order."""
    with torch.no_grad():
        x2 = _x_rows(x, "x")
        R, D = x2.shape
        dev = x2.device
        if grad.shape != x.shape or grad.dtype != x.dtype or grad.device != dev:
            raise ValueError("grad must match x in shape, dtype and device")
        g2 = _x_rows(grad, "grad")
        mean, rstd = stats
        for t in (mean, rstd):
            if t.shape != (R,) or t.dtype != torch.float32 or t.device != dev or not t.is_contiguous():
                raise ValueError(f"stats must be the forward call's: two float32 [{R}] tensors")
        w, b = _affine(weight, x, "weight"), _affine(bias, x, "bias")
        dx = torch.empty(x.shape, dtype=x.dtype, device=dev) if need_dx else None
        dw = torch.empty_like(w) if need_dweight and w is not None else None
        db = torch.empty_like(b) if need_dbias and b is not None else None
        a = NormGradArgs()
        a.struct_size = ctypes.sizeof(NormGradArgs)
        a.dtype, a.wdtype = _DTYPES[x2.dtype], _wdtype(x2, w, b)
        a.x, a.rows, a.dim, a.ld = x2.data_ptr(), R, D, x2.stride(0) if R > 1 else D
        a.weight, a.grad, a.grad_ld = ptr(w), g2.data_ptr(), g2.stride(0) if R > 1 else D
        a.mean, a.rstd = mean.data_ptr(), rstd.data_ptr()
        a.out_dx, a.out_ld, a.out_dweight, a.out_dbias = ptr(dx), D, ptr(dw), ptr(db)
        ws = None
        if dw is not None or db is not None:
            n = _workspace_bytes(R, D, a.dtype)
            ws = torch.empty(n, dtype=torch.uint8, device=dev)
            a.workspace, a.workspace_bytes = ws.data_ptr(), n
        if dx is not None or ws is not None:
            call(lib().fl_layer_norm_grad, a, dev, "fl_layer_norm_grad")
        return dx, dw, db


@lru_cache(maxsize=256)
def _workspace_bytes(rows: int, dim: int, dtype: int) -> int:
    n = ctypes.c_size_t(0)
    _lib.check(lib().fl_layer_norm_grad_workspace_bytes(rows, dim, dtype, ctypes.byref(n)),
               "fl_layer_norm_grad_workspace_bytes")
    return n.value
