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

from typing import Optional, Tuple

import torch

from . import _lib

_CACHE_DTYPES = (torch.bfloat16, torch.float16, torch.float8_e4m3fn)


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
        _lib.autograd().check_cache(k, v, k_scale, v_scale)
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


def cache_write(cache: PagedCache, k: torch.Tensor, v: torch.Tensor, table: torch.Tensor, lengths: torch.Tensor, *,
                starts: Optional[torch.Tensor] = None) -> None:
    """Write new tokens' keys and values ``[..., heads, dim]`` (the leading dimensions
    are the call's rows; any strides) into the cache: in its dtype as they are, or
    from float32, bfloat16 or float16 in 8 bits with a scale for each token and head.
    One launch.  Sequences that share pages must not write the same slot in a call."""
    _check_cache(cache)
    _lib.autograd().cache_write(cache.k, cache.v, cache.k_scale, cache.v_scale, k, v, table, lengths, starts)


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
    out_k, out_v = out if out is not None else (None, None)
    return _lib.autograd().cache_read(cache.k, cache.v, cache.k_scale, cache.v_scale, table, lengths, tokens, starts, dtype, out_k,
                                      out_v)


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
    result has its dtype and shape, in ``out`` where given (``q`` itself, or memory apart
    from it; rows behind the last sequence stay as they were; without ``out`` they hold
    anything).  With
    ``return_lse`` also the float32 log-sum-exp ``[..., q_heads]`` of each row's scores.

    A token that sees nothing has 0 and -inf, one all of whose scores are -inf NaN (0 / 0)
    and -inf.  What a slot holds that a token does
    not see, NaN and infinity included, has no part in its result; values seen are
    taken up to 2^100 in magnitude.  Sums in float32; the weights are rounded
    for the product with the values: to ``q``'s dtype, over 8 bits (where they carry
    their values' scales) to bfloat16.  15 bits of them are kept, so that the result's own
    rounding is what is left, for float16 queries over 8 bits, and for bfloat16 ones of
    ``dim`` up to 128 where a sequence has up to 32 rows (new tokens times query heads per
    cached head; 64 over 8 bits): decode and verify steps.
    One to three launches (with ``starts`` one for each kind of sequence, and the joining
    of split ones), without host synchronisation; results are the same each
    time, and depend on how the call's shapes split the keys in the last bits."""
    _check_cache(cache)
    o, lse = _lib.autograd().attention(cache.k, cache.v, cache.k_scale, cache.v_scale, q, table, lengths, starts, scale, softcap,
                                       window, sinks, out, return_lse)
    o = out if out is not None else o
    return (o, lse) if return_lse else o
