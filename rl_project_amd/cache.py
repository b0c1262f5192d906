"""A paged key / value cache on the device, and attention over it: what a decode or
verify step's layers do between the projections (reference ``models/attention/`` on
the caches that ``inference/engine.py:141-161`` merges per step, with the pages that
``inference/paged_memory.py:22`` accounts for on the host).

The tokens of a call.  Every call names them by the same three device tensors, read
by the kernels (no host synchronisation, so a captured step may update them):

``table``    int32 ``[B, width]``: page numbers; position ``t`` of sequence ``b`` is
             slot ``t % page_size`` of page ``table[b, t // page_size]``
``lengths``  int32 ``[B]``: the tokens each sequence has, the call's new ones among them
``starts``   int32 ``[B + 1]``, ascending from 0: rows ``starts[b]`` to ``starts[b + 1] -
             1`` of the call's tensors are sequence ``b``'s newest tokens, the last one
             at position ``lengths[b] - 1``.  None: every sequence has as many (the rows
             over ``B``; a decode step has one each).

Rows behind the last sequence (a padded batch's) are left as they were.  A position
below 0 is no token; a page number outside the cache, or a position past the table, is
a missing page: such a token is not written, reads as NaN, and gives NaN to the tokens
that would see it."""

from __future__ import annotations

import math
from typing import List, Optional, Sequence, Tuple

import torch

from . import _lib

_PAGE_SIZES = (16, 32, 64, 128)
_CACHE_DTYPES = (torch.bfloat16, torch.float16, torch.float8_e4m3fn)
_ROW_DTYPES = (torch.float32, torch.bfloat16, torch.float16)


class PagedCache:
    """One layer's keys and values in pages: ``k [pages, heads, page_size, dim]`` and
    ``v [pages, heads, dim, page_size]`` (a channel's tokens side by side, as the
    matrix cores read them), contiguous, ``page_size`` 16, 32, 64 or 128, ``dim`` a
    multiple of 8 up to 256.

    bfloat16, float16, or float8_e4m3fn with ``k_scale`` and ``v_scale`` (uint8
    ``[pages, heads, page_size]``): a value of the last stands for itself times
    ``2 ** (scale - 127)``, the least power of two that takes the token's largest
    finite magnitude in that head to 448 or below (from 2^-96 to 2^120), so that
    quantising rounds once, to 3 bits behind the leading one.  NaN and infinity are
    stored as NaN.

    ``PagedCache.empty(...)`` allocates; the tensors may also be a caller's own."""

    __slots__ = ("k", "v", "k_scale", "v_scale")

    def __init__(self, k: torch.Tensor, v: torch.Tensor, k_scale: Optional[torch.Tensor] = None,
                 v_scale: Optional[torch.Tensor] = None):
        if k.device.type != "cuda":
            raise ValueError("the cache must be on a ROCm device (no CPU fallback)")
        if k.dim() != 4 or v.dim() != 4 or v.shape != (k.size(0), k.size(1), k.size(3), k.size(2)):
            raise ValueError(f"k [pages, heads, page_size, dim] and v [pages, heads, dim, page_size] do not match: "
                             f"{tuple(k.shape)}, {tuple(v.shape)}")
        if k.dtype not in _CACHE_DTYPES:
            raise NotImplementedError(f"cache dtype {k.dtype} is not supported (bfloat16, float16, float8_e4m3fn)")
        if v.dtype != k.dtype or v.device != k.device or not k.is_contiguous() or not v.is_contiguous():
            raise ValueError("k and v must share a dtype and a device and be contiguous")
        pages, heads, page_size, dim = k.shape
        if page_size not in _PAGE_SIZES:
            raise ValueError(f"page_size {page_size} is none of {_PAGE_SIZES}")
        if pages < 1 or heads < 1 or dim < 8 or dim % 8 or dim > _lib.FL_CACHE_MAX_DIM:
            raise ValueError(f"{pages} pages, {heads} heads, dim {dim}: at least one of each, dim a multiple of 8 up to "
                             f"{_lib.FL_CACHE_MAX_DIM}")
        if k.dtype == torch.float8_e4m3fn:
            for s in (k_scale, v_scale):
                if s is None or s.dtype != torch.uint8 or s.shape != k.shape[:3] or s.device != k.device or not s.is_contiguous():
                    raise ValueError(f"a float8_e4m3fn cache needs k_scale and v_scale: contiguous uint8 {tuple(k.shape[:3])}")
        elif k_scale is not None or v_scale is not None:
            raise ValueError("scales belong to a float8_e4m3fn cache")
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale

    @classmethod
    def empty(cls, pages: int, heads: int, dim: int, *, page_size: int = 64, dtype: torch.dtype = torch.bfloat16,
              device="cuda") -> "PagedCache":
        """A cache of zeros."""
        if dtype not in _CACHE_DTYPES:
            raise NotImplementedError(f"cache dtype {dtype} is not supported (bfloat16, float16, float8_e4m3fn)")
        k = torch.zeros(pages, heads, page_size, dim, dtype=dtype, device=device)
        v = torch.zeros(pages, heads, dim, page_size, dtype=dtype, device=device)
        if dtype != torch.float8_e4m3fn:
            return cls(k, v)
        return cls(k, v, *(torch.full((pages, heads, page_size), 127, dtype=torch.uint8, device=device) for _ in "kv"))

    @property
    def pages(self) -> int:
        return self.k.size(0)

    @property
    def heads(self) -> int:
        return self.k.size(1)

    @property
    def page_size(self) -> int:
        return self.k.size(2)

    @property
    def dim(self) -> int:
        return self.k.size(3)

    @property
    def dtype(self) -> torch.dtype:
        return self.k.dtype

    @property
    def device(self) -> torch.device:
        return self.k.device


def _check_cache(cache) -> None:
    if not isinstance(cache, PagedCache):
        raise TypeError("cache must be a PagedCache")


def _check_tokens(cache: PagedCache, table: torch.Tensor, lengths: torch.Tensor, starts: Optional[torch.Tensor], rows: int) -> None:
    dev = cache.k.device
    if table.dim() != 2 or table.dtype != torch.int32 or table.device != dev or (table.size(1) > 1 and table.stride(1) != 1):
        raise ValueError(f"table must be int32 [B, width] on {dev}, its rows contiguous")
    B = table.size(0)
    if lengths.shape != (B,) or lengths.dtype != torch.int32 or lengths.device != dev or not lengths.is_contiguous():
        raise ValueError(f"lengths must be contiguous int32 [{B}] on {dev}")
    if starts is None:
        if (B and rows % B) or (rows and not B):
            raise ValueError(f"{rows} tokens are not as many for each of {B} sequences: give starts")
    elif starts.shape != (B + 1,) or starts.dtype != torch.int32 or starts.device != dev or not starts.is_contiguous():
        raise ValueError(f"starts must be contiguous int32 [{B + 1}] on {dev}")


def _check_rows(cache: PagedCache, x: torch.Tensor, name: str, heads: Optional[int] = None) -> None:
    if x.dim() < 3 or x.size(-1) != cache.dim or (heads is not None and x.size(-2) != heads) or x.device != cache.device:
        raise ValueError(f"{name} must be [..., {heads if heads is not None else 'heads'}, {cache.dim}] on {cache.device}, "
                         f"not {tuple(x.shape)}")


def _no_gradient(what: str, *tensors: torch.Tensor) -> None:
    if torch.is_grad_enabled() and any(t.requires_grad for t in tensors):
        raise RuntimeError(f"{what} records no gradient: call it under torch.no_grad()")


def cache_write(cache: PagedCache, k: torch.Tensor, v: torch.Tensor, table: torch.Tensor, lengths: torch.Tensor, *,
                starts: Optional[torch.Tensor] = None) -> None:
    """Write new tokens' keys and values ``[..., heads, dim]`` (the leading dimensions
    are the call's rows; any strides) into the cache: in its dtype as they are, or
    from float32, bfloat16 or float16 in 8 bits with a scale for each token and head.
    One launch.  Sequences that share pages must not write the same slot in a call."""
    _check_cache(cache)
    _check_rows(cache, k, "k", cache.heads)
    if v.shape != k.shape or v.dtype != k.dtype or v.device != k.device:
        raise ValueError("k and v must match in shape, dtype and device")
    if k.dtype not in _ROW_DTYPES or (cache.dtype != torch.float8_e4m3fn and k.dtype != cache.dtype):
        raise NotImplementedError(f"{k.dtype} keys into a {cache.dtype} cache")
    _check_tokens(cache, table, lengths, starts, k.shape[:-2].numel())
    _no_gradient("cache_write", k, v)
    _lib.autograd().cache_call(cache.k, cache.v, cache.k_scale, cache.v_scale, k, v, table, lengths, starts, True)


def cache_read(cache: PagedCache, table: torch.Tensor, lengths: torch.Tensor, tokens: int, *, starts: Optional[torch.Tensor] = None,
               dtype: Optional[torch.dtype] = None, out: Optional[Tuple[torch.Tensor, torch.Tensor]] = None
               ) -> Tuple[torch.Tensor, torch.Tensor]:
    """``(k, v)``, each ``[tokens, heads, dim]``: what the cache holds of each
    sequence's newest tokens, named as for ``cache_write`` (all of a sequence's where
    ``starts`` gives it as many rows as it has tokens), in ``dtype`` (the cache's, or
    float32 for 8 bits): exact but for one rounding to a 16-bit ``dtype`` of values
    outside its range.  Into ``out`` (contiguous) where given (rows behind the
    last sequence stay as they were; without ``out`` they hold anything).  One launch."""
    _check_cache(cache)
    if out is not None:
        dtype = out[0].dtype
    elif dtype is None:
        dtype = torch.float32 if cache.dtype == torch.float8_e4m3fn else cache.dtype
    if dtype not in _ROW_DTYPES:
        raise NotImplementedError(f"dtype {dtype} is not supported (float32, bfloat16, float16)")
    if tokens < 0:
        raise ValueError(f"tokens {tokens} < 0")
    _check_tokens(cache, table, lengths, starts, tokens)
    shape = (tokens, cache.heads, cache.dim)
    if out is None:
        out = tuple(torch.empty(shape, dtype=dtype, device=cache.device) for _ in range(2))
    elif any(t.shape != shape or t.dtype != dtype or t.device != cache.device or not t.is_contiguous() for t in out):
        raise ValueError(f"out must be two contiguous {dtype} tensors {shape} on {cache.device}")
    _lib.autograd().cache_call(cache.k, cache.v, cache.k_scale, cache.v_scale, out[0], out[1], table, lengths, starts, False)
    return out[0], out[1]


def paged_attention(q: torch.Tensor, cache: PagedCache, table: torch.Tensor, lengths: torch.Tensor, *,
                    starts: Optional[torch.Tensor] = None, scale: Optional[float] = None, window: Optional[int] = None,
                    sinks: int = 0, softcap: float = 0.0, return_lse: bool = False, out: Optional[torch.Tensor] = None):
    """Attention of each sequence's newest tokens, ``q [..., q_heads, dim]``, over all
    it has in the cache (their own keys and values among them: ``cache_write`` first):

        ``softmax(softcap * tanh(scale * q . k / softcap)) v``   (softcap 0: ``scale * q . k``)

    over positions ``t <= p`` of a token at position ``p``; with ``window`` only ``t > p -
    window`` and the first ``sinks`` positions.  ``q_heads`` is a multiple of the
    cache's ``heads``, neighbouring query heads share one; ``scale`` is 1 / sqrt(dim)
    where not given.  ``q`` is bfloat16 or float16, a 16-bit cache's own dtype; the
    result has its dtype and shape, in ``out`` where given (rows behind the last
    sequence stay as they were; without ``out`` they hold anything).  With
    ``return_lse`` also the float32 log-sum-exp ``[..., q_heads]`` of each row's scores.

    A token that sees nothing has 0 and -inf.  What a slot holds that a token does
    not see, NaN and infinity included, has no part in its result; values seen are
    taken up to 2^100 in magnitude.  Sums in float32; the weights are rounded once
    to ``q``'s dtype (bfloat16 over an 8-bit cache) for the product with the values.
    One or two launches, without host synchronisation; results are the same each
    time, and depend on how the call's shapes split the keys in the last bits."""
    _check_cache(cache)
    _check_rows(cache, q, "q")
    if q.dtype not in (torch.bfloat16, torch.float16) or (cache.dtype != torch.float8_e4m3fn and q.dtype != cache.dtype):
        raise NotImplementedError(f"{q.dtype} queries over a {cache.dtype} cache")
    if q.size(-2) < 1 or q.size(-2) % cache.heads:
        raise ValueError(f"{q.size(-2)} query heads over {cache.heads} cached")
    _check_tokens(cache, table, lengths, starts, q.shape[:-2].numel())
    if scale is None:
        scale = 1.0 / math.sqrt(cache.dim)
    window = 0 if window is None else window
    if window < 0 or sinks < 0:
        raise ValueError("window and sinks must be >= 0")
    _no_gradient("paged_attention", q)
    into = None
    if out is not None:
        if out.shape != q.shape or out.dtype != q.dtype or out.device != q.device:
            raise ValueError("out must match q in shape, dtype and device")
        into = out if out.dim() == 3 else out.view(-1, out.size(-2), out.size(-1))
        if into.data_ptr() % 8 or into.stride(2) != 1 or any(
                into.size(i) > 1 and (into.stride(i) % 4 or into.stride(i) < cache.dim) for i in (0, 1)):
            raise ValueError("out must be 8-byte aligned, its heads contiguous and apart, strides in multiples of 4 elements")
    o, lse = _lib.autograd().attention(cache.k, cache.v, cache.k_scale, cache.v_scale, q, table, lengths, starts, scale, softcap,
                                       window, sinks, into, return_lse)
    o = out if out is not None else o
    return (o, lse) if return_lse else o
