"""Norms of queries and keys for each head and their rotation by position, in one
pass, with gradients; and the frequencies of the rotation.

The model in front of the sampler (reference ``models/attention/``; its rotation
takes scalings for long contexts, ``core/config.py:49-56``) computes them as
several tensor operations."""

from __future__ import annotations

import math
from typing import Optional, Tuple

import torch

from . import _lib


def rotary_frequencies(dim: int, base: float = 10000.0, *, scaling: Optional[str] = None, factor: float = 1.0,
                       original_length: Optional[int] = None, device=None) -> Tuple[torch.Tensor, float]:
    """``(inv_freq, gain)`` of a rotation of ``dim`` values (even): float64 ``[dim / 2]``
    angles per position, ``base ** (-2 p / dim)``, and the factor on the rotated values.

    ``scaling`` stretches them for contexts ``factor`` times as long as the model
    was trained on (``original_length`` positions):

    * ``"linear"``: every frequency over ``factor`` (position interpolation,
      Chen et al., arXiv:2306.15595).
    * ``"ntk"``: ``base * factor ** (dim / (dim - 2))``, which leaves the highest
      frequency as it is and divides the lowest by ``factor``.
    * ``"yarn"``: pairs that turn more than 32 times over ``original_length`` as
      they are, fewer than once over ``factor``, a line between them in the pair's
      number; gain ``0.1 ln factor + 1`` (Peng et al., arXiv:2309.00071)."""
    if dim < 2 or dim % 2:
        raise ValueError(f"dim must be even and at least 2, not {dim}")
    if not (base > 1.0 and math.isfinite(base)) or not (factor >= 1.0 and math.isfinite(factor)):
        raise ValueError("base must be above 1 and factor at least 1")
    at = torch.arange(0, dim, 2, dtype=torch.float64) / dim
    gain = 1.0
    if scaling == "ntk":
        if dim < 4:
            raise ValueError("ntk scaling needs dim of at least 4")
        base = base * factor ** (dim / (dim - 2))
    inv = float(base) ** -at
    if scaling == "linear":
        inv = inv / factor
    elif scaling == "yarn":
        if not original_length or original_length < 1:
            raise ValueError("yarn scaling needs original_length")
        # the pair that turns `turns` times over the original length
        pair = lambda turns: dim * math.log(original_length / (turns * 2 * math.pi)) / (2 * math.log(base))  # noqa: E731
        low, high = max(math.floor(pair(32.0)), 0), min(math.ceil(pair(1.0)), dim - 1)
        ramp = ((torch.arange(dim // 2, dtype=torch.float64) - low) / max(high - low, 1e-3)).clamp(0, 1)
        if pair(1.0) < 0:   # (none turns once)
            ramp.fill_(1.0)
        inv = inv * (1 - ramp) + inv / factor * ramp
        gain = 0.1 * math.log(factor) + 1.0
    elif scaling not in (None, "ntk"):
        raise ValueError(f"scaling {scaling!r} is none of linear, ntk, yarn")
    return inv.to(device) if device is not None else inv, gain


def qk_norm_rope(q: torch.Tensor, k: torch.Tensor, positions: torch.Tensor, inv_freq: torch.Tensor, *,
                 q_weight: Optional[torch.Tensor] = None, k_weight: Optional[torch.Tensor] = None, eps: Optional[float] = None,
                 interleaved: bool = False, gain: float = 1.0) -> Tuple[torch.Tensor, torch.Tensor]:
    """Queries ``[..., heads, D]`` and keys ``[..., kv_heads, D]``, each head normed
    and rotated by its token's position, in one pass: with ``eps`` the norm
    ``y = x / sqrt(mean(x^2) + eps) * weight`` over ``D`` (weights ``[D]``, None: 1, of
    one dtype, ``q``'s or float32), without it ``y = x``; then the first
    ``2 * len(inv_freq)`` values of ``y`` turned in pairs, pair ``p`` by ``position *
    inv_freq[p]`` and ``gain``: values ``p`` and ``p + len(inv_freq)``, or with
    ``interleaved`` ``2 p`` and ``2 p + 1``.

    ``positions`` (int32 or int64, any sign) has the leading dimensions, or expands
    to them; ``inv_freq`` is float64 or float32 (``rotary_frequencies``).  Float32,
    bfloat16 or float16, ``D`` even up to 512; ``q`` and ``k`` may be strided (views of
    one projection's output); the results are contiguous.  Sums in float32, angles in
    float64, one rounding at the end.

    Differentiable (once, in reverse mode) in ``q``, ``k`` and the weights (an ``inv_freq``
    that requires a gradient is refused where one would be recorded), except
    under stream capture: a captured step takes this call under ``torch.no_grad()``
    and ``qk_norm_rope_backward``."""
    out = _lib.autograd().qk_norm_rope(q, k, positions, inv_freq, q_weight, k_weight, eps, interleaved, gain)
    return out[0], out[1]


def qk_norm_rope_backward(grad_q: Optional[torch.Tensor], grad_k: Optional[torch.Tensor], q: torch.Tensor, k: torch.Tensor,
                          positions: torch.Tensor, inv_freq: torch.Tensor, *, q_weight: Optional[torch.Tensor] = None,
                          k_weight: Optional[torch.Tensor] = None, eps: Optional[float] = None, interleaved: bool = False,
                          gain: float = 1.0, need_dweight: bool = True):
    """``(dq, dk, dq_weight, dk_weight)`` of ``qk_norm_rope`` for upstream gradients of
    its results (either may be None, and so are its side's then): what autograd
    computes, as launches that a graph may record.  ``q`` and ``k`` are the forward
    call's inputs.  The weights' gradients (None without a weight) have their dtype;
    their sums over tokens and heads have a fixed order."""
    return tuple(_lib.autograd().qk_norm_rope_backward(grad_q, grad_k, q, k, positions, inv_freq, q_weight, k_weight, eps,
                                                       interleaved, gain, need_dweight))
