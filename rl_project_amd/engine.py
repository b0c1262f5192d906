"""Batched decode-group sampling with device-resident state: the replacement
for ``InferenceEngine._emit``'s per-request loop (reference
``inference/engine.py:114-139``, called per sequence from ``_decode_group``,
``:141-160``).

The reference samples each sequence of a decode group separately:
``apply_sampling_filters`` + ``sample_from_logits`` on a ``[1, V]`` slice and
``.item()`` per sequence, with the sequence's prompt + generated ids as the
penalty history (``engine.py:40,118-122``) and ``stop_token_ids`` plus the
EOS id as its stop set (``engine.py:123-125``).

``BatchedSampler`` keeps all of that on the device, per slot:

* the sampling parameters as arrays;
* the history ids, with capacity ``max_seq_len``;
* the stop set.

``step(logits)`` samples every row in one launch; the kernel also sets the
finished flags and appends the tokens to the histories (no host
synchronisation, no other kernel). It returns device tensors; the caller
reads them back once per step, not once per sequence. Length limits,
cancellation and block allocation stay with the engine, as in the reference.

``CacheGroup`` is the group's other state: its layers' keys and values in pages
(the reference merges per-sequence caches each step, ``engine.py:146-150``, and
accounts for blocks on the host, ``inference/paged_memory.py:22``).
"""

from __future__ import annotations

from typing import Dict, Iterable, List, Optional, Sequence, Tuple

import torch

from .cache import PagedCache, cache_write, paged_attention
from .params import SamplingParams
from . import _lib
from .sampling import SampleOutput, _Call, _check_logits


class BatchedSampler:
    """Device-resident sampling state of up to ``max_rows`` sequences.

    Row ``i`` of a step's logits belongs to slot ``i`` (or to ``slots[i]`` when
    the step names its slots); ``admit`` / ``release`` manage which request
    holds which slot.  A step is one ``fl_sample`` launch: the kernel samples
    every row, sets the finished flags in place and appends each token to its
    slot's history (``FL_FLAG_APPEND_HISTORY``); nothing is synchronised with
    the host and nothing is allocated (the argument block and the output
    buffers are kept per row count and reused, so a step's outputs are valid
    until the next step)."""

    def __init__(self, max_rows: int, max_seq_len: int, vocab: int, device, *, eos_token_id: Optional[int] = None,
                 max_stop_ids: int = 8, generator: Optional[torch.Generator] = None):
        self.max_rows, self.max_seq_len, self.vocab = max_rows, max_seq_len, vocab
        self.device = torch.device(device)
        self.eos = eos_token_id
        self.generator = generator
        d = self.device
        self.temperature = torch.ones(max_rows, dtype=torch.float32, device=d)
        self.top_k = torch.zeros(max_rows, dtype=torch.int32, device=d)
        self.top_p = torch.ones(max_rows, dtype=torch.float32, device=d)
        self.min_p = torch.zeros(max_rows, dtype=torch.float32, device=d)
        self.rep_penalty = torch.ones(max_rows, dtype=torch.float32, device=d)
        self.history = torch.full((max_rows, max_seq_len), -1, dtype=torch.int32, device=d)
        self.hist_len = torch.zeros(max_rows, dtype=torch.int32, device=d)
        self.stop_ids = torch.full((max_rows, max_stop_ids + 1), -1, dtype=torch.int32, device=d)
        # uint8, updated in place by the kernel (finished_in and out_finished)
        self.finished_u8 = torch.ones(max_rows, dtype=torch.uint8, device=d)
        self._plans: Dict[Tuple[int, torch.dtype, int, int, bool], _Call] = {}

    @property
    def finished(self) -> torch.Tensor:
        """bool [max_rows]: slots that produced a stop id or were released."""
        return self.finished_u8.view(torch.bool)

    def admit(self, slot: int, params: SamplingParams, prompt_tokens: Sequence[int]) -> None:
        """Give ``slot`` to a new request: its parameters (validated as
        ``requests.py:33-41``), its prompt as the start of its history and its
        stop set (``stop_token_ids`` plus the EOS id)."""
        params.validate()
        n = len(prompt_tokens)
        if n >= self.max_seq_len:
            raise ValueError(f"prompt of {n} tokens does not fit max_seq_len {self.max_seq_len}")
        stops = sorted(set(int(s) for s in params.stop_token_ids) | ({self.eos} if self.eos is not None else set()))
        if len(stops) > self.stop_ids.size(1):
            raise ValueError(f"{len(stops)} stop ids exceed the {self.stop_ids.size(1)} slots per row")
        if any(t < 0 or t >= self.vocab for t in prompt_tokens):
            raise IndexError("prompt token outside the vocabulary")
        self.temperature[slot] = float(params.temperature)
        self.top_k[slot] = int(params.top_k or 0)
        self.top_p[slot] = float(params.top_p if params.top_p is not None else 1.0)
        self.min_p[slot] = float(params.min_p or 0.0)
        self.rep_penalty[slot] = float(params.repetition_penalty)
        row = torch.full((self.max_seq_len,), -1, dtype=torch.int32)
        row[:n] = torch.tensor(list(prompt_tokens), dtype=torch.int32)
        self.history[slot].copy_(row, non_blocking=False)
        self.hist_len[slot] = n
        srow = torch.full((self.stop_ids.size(1),), -1, dtype=torch.int32)
        if stops:
            srow[:len(stops)] = torch.tensor(stops, dtype=torch.int32)
        self.stop_ids[slot].copy_(srow)
        self.finished_u8[slot] = 0

    def release(self, slot: int) -> None:
        """Retire ``slot``: it is finished (a row of a later step that still
        maps to it samples but appends nothing) and its history is emptied."""
        self.finished_u8[slot] = 1
        self.hist_len[slot] = 0

    def _plan(self, n: int, logits: torch.Tensor, want_logprob: bool) -> _Call:
        key = (n, logits.dtype, logits.size(1), logits.stride(0), want_logprob)
        call = self._plans.get(key)
        if call is None:
            call = _Call(logits, temperature=self.temperature[:n], top_k=self.top_k[:n], top_p=self.top_p[:n],
                         min_p=self.min_p[:n], repetition_penalty=self.rep_penalty[:n],
                         history=(self.history[:n], self.hist_len[:n]), stop_ids=self.stop_ids[:n],
                         uniforms=torch.zeros(n, dtype=torch.float32, device=self.device),
                         finished=self.finished_u8[:n], out_finished=self.finished_u8[:n],
                         flags=_lib.FL_FLAG_APPEND_HISTORY, want_logprob=want_logprob)
            # the state tensors are used in place, never copied
            assert call.hist.data_ptr() == self.history.data_ptr() and call.fin_in.data_ptr() == \
                self.finished_u8.data_ptr()
            self._plans[key] = call
        return call

    def step(self, logits: torch.Tensor, uniforms: Optional[torch.Tensor] = None, return_logprobs: bool = False,
             slots: Optional[torch.Tensor] = None) -> SampleOutput:
        """Sample one token for each row of ``logits`` (row i: slot i, or
        ``slots[i]``), mark the rows that produced a stop id as finished and
        append the tokens of unfinished rows to their histories, in one launch
        with no host synchronisation.  ``status`` of the output carries the
        per-row FL_ROW_* bits for the caller to read with the tokens."""
        n = logits.size(0)
        if n > self.max_rows:
            raise ValueError(f"{n} rows exceed max_rows {self.max_rows}")
        if uniforms is None:
            uniforms = torch.rand(n, device=self.device, generator=self.generator)
        if slots is not None:
            return self._step_slots(logits, uniforms, return_logprobs, slots)
        logits = _check_logits(logits)
        call = self._plan(n, logits, return_logprobs)
        if uniforms.dtype != torch.float32 or not uniforms.is_contiguous() or uniforms.numel() != n:
            raise ValueError("uniforms must be a contiguous float32 tensor with one draw per row")
        call.args.logits = logits.data_ptr()
        call.args.uniforms = uniforms.data_ptr()
        call.keep = (logits, uniforms)   # alive until the kernel has read them
        call.run_exact()
        return SampleOutput(call.tokens, call.finished[:n].view(torch.bool), call.status, call.logprob)

    def _step_slots(self, logits, uniforms, return_logprobs, slots) -> SampleOutput:
        """A decode group whose rows map to arbitrary slots: gather the slots'
        state, sample with the append, scatter the state back (a few small
        device copies; no host synchronisation)."""
        idx = slots.to(device=self.device, dtype=torch.long)
        hist = self.history.index_select(0, idx)
        hlen = self.hist_len.index_select(0, idx)
        fin = self.finished_u8.index_select(0, idx)
        call = _Call(logits, temperature=self.temperature[idx], top_k=self.top_k[idx], top_p=self.top_p[idx],
                     min_p=self.min_p[idx], repetition_penalty=self.rep_penalty[idx], history=(hist, hlen),
                     stop_ids=self.stop_ids[idx], uniforms=uniforms, finished=fin, out_finished=fin,
                     flags=_lib.FL_FLAG_APPEND_HISTORY, want_logprob=return_logprobs).run_exact()
        self.history.index_copy_(0, idx, hist)
        self.hist_len.index_copy_(0, idx, hlen)
        self.finished_u8.index_copy_(0, idx, fin)
        return SampleOutput(call.tokens, fin.view(torch.bool), call.status, call.logprob)

    def history_of(self, slot: int) -> List[int]:
        """Prompt + generated ids of a slot (reads the device: for tests and retirement)."""
        return self.history[slot, : int(self.hist_len[slot])].tolist()


class CacheFull(RuntimeError):
    """No pages left for a step's new tokens (the step changed nothing)."""


class CacheStep:
    """The new tokens of one step over a ``CacheGroup``, as its layers take them:
    rows ``starts[i]`` to ``starts[i + 1] - 1`` of a layer's tensors are slot ``slots[i]``'s,
    oldest first; ``positions`` (int64 ``[tokens]``) are theirs, for ``qk_norm_rope``.
    ``table``, ``lengths`` and ``starts`` (None where every slot has as many tokens) are
    what ``cache_write`` and ``paged_attention`` take."""

    __slots__ = ("layers", "slots", "counts", "tokens", "table", "lengths", "starts", "positions")

    def __init__(self, layers, slots, counts, table, lengths, starts, positions):
        self.layers, self.slots, self.counts = layers, slots, counts
        self.tokens = sum(counts)
        self.table, self.lengths, self.starts, self.positions = table, lengths, starts, positions

    def attend(self, layer: int, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, **kw) -> torch.Tensor:
        """A layer's attention of the step: its new keys and values into the cache, its
        queries over all that the sequences have there (``paged_attention``'s keywords)."""
        cache = self.layers[layer]
        cache_write(cache, k, v, self.table, self.lengths, starts=self.starts)
        return paged_attention(q, cache, self.table, self.lengths, starts=self.starts, **kw)


class CacheGroup:
    """The paged caches of up to ``max_rows`` sequences: one ``PagedCache`` per layer,
    of one shape, whose pages all layers number alike.

    ``step(slots, counts)`` makes room for each slot's new tokens (pages are taken as
    they are needed) and names them for the layers; ``truncate`` takes a slot's newest
    tokens back (rejected drafts) and ``release`` all of them.  Page numbers and lengths
    live on the host; a step sends them in one copy, as new tensors whose table is as wide
    as its longest slot needs.  (A captured step takes a table, lengths and starts of fixed
    places, which the program writes before each replay, straight to ``cache_write`` and
    ``paged_attention``.)"""

    def __init__(self, layers: Sequence[PagedCache], max_rows: int, max_seq_len: int):
        layers = list(layers)
        if not layers or any(not isinstance(c, PagedCache) for c in layers):
            raise TypeError("layers must be PagedCaches, one at least")
        if any((c.pages, c.page_size, c.device) != (layers[0].pages, layers[0].page_size, layers[0].device) for c in layers):
            raise ValueError("the layers' caches must have as many pages, of one size, on one device")
        if max_rows < 1 or max_seq_len < 1:
            raise ValueError("max_rows and max_seq_len must be at least 1")
        self.layers = layers
        self.max_rows, self.max_seq_len = max_rows, max_seq_len
        self.page_size, self.device = layers[0].page_size, layers[0].device
        self._free = list(range(layers[0].pages - 1, -1, -1))
        self._pages: List[List[int]] = [[] for _ in range(max_rows)]
        self._lens = [0] * max_rows

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def length(self, slot: int) -> int:
        """Tokens that the slot has in the cache."""
        return self._lens[self._slot(slot)]

    def _slot(self, slot: int) -> int:
        if not 0 <= slot < self.max_rows:
            raise IndexError(f"slot {slot} outside 0 .. {self.max_rows - 1}")
        return slot

    def step(self, slots: Sequence[int], counts: Sequence[int]) -> CacheStep:
        """Room for ``counts[i]`` new tokens of slot ``slots[i]`` (each slot once), which
        count as cached from here on.  ``CacheFull`` where the pages do not suffice.  A
        step that raises changed nothing."""
        slots, counts = [int(s) for s in slots], [int(c) for c in counts]
        if not slots or len(slots) != len(counts) or len(set(slots)) != len(slots):
            raise ValueError("slots must differ, with a count each, one at least")
        if any(s < 0 or s >= self.max_rows for s in slots):
            raise IndexError(f"a slot outside 0 .. {self.max_rows - 1}")
        if any(c < 1 for c in counts):
            raise ValueError("every slot of a step needs at least one new token")
        need = []
        for s, c in zip(slots, counts):
            n = self._lens[s] + c
            if n > self.max_seq_len:
                raise ValueError(f"slot {s}: {n} tokens exceed max_seq_len {self.max_seq_len}")
            need.append(-(-n // self.page_size) - len(self._pages[s]))
        if sum(need) > len(self._free):
            raise CacheFull(f"{sum(need)} pages needed, {len(self._free)} free")
        B, N = len(slots), sum(counts)
        left = len(self._free)
        pages: List[List[int]] = []
        for s, n in zip(slots, need):
            pages.append(self._pages[s] + self._free[left - n: left][::-1])
            left -= n
        width = max(map(len, pages))
        flat: List[int] = []
        for p in pages:
            flat += p + [-1] * (width - len(p))
        flat += [self._lens[s] + c for s, c in zip(slots, counts)]
        at = [0]
        for c in counts:
            at.append(at[-1] + c)
        flat += at
        sent = torch.tensor(flat, dtype=torch.int32).to(self.device)
        table, lengths, starts = sent[: B * width].view(B, width), sent[B * width: B * width + B], sent[B * width + B:]
        ends = starts[1:]
        row = torch.arange(N, dtype=torch.int32, device=self.device)
        if len(set(counts)) == 1:
            positions = ((lengths - ends)[:, None] + row.view(B, -1)).view(-1).to(torch.int64)
            starts = None
        else:
            positions = (row + (lengths - ends)[torch.searchsorted(ends, row, right=True)]).to(torch.int64)
        # (from here on nothing can fail)
        del self._free[left:]
        for s, c, p in zip(slots, counts, pages):
            self._pages[s] = p
            self._lens[s] += c
        return CacheStep(self.layers, slots, counts, table, lengths, starts, positions)

    def truncate(self, slot: int, length: int) -> None:
        """Keep the slot's first ``length`` tokens; pages without any are free again."""
        if not 0 <= length <= self._lens[self._slot(slot)]:
            raise ValueError(f"length {length} outside 0 .. {self._lens[slot]}")
        keep = -(-length // self.page_size)
        self._free += reversed(self._pages[slot][keep:])
        del self._pages[slot][keep:]
        self._lens[slot] = length

    def release(self, slot: int) -> None:
        """Free all of the slot's pages."""
        self.truncate(slot, 0)
