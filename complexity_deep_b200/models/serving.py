"""Decode steps of sequences with lengths of their own: a captured step over a paged cache, from one token per slot to the next one,
drawn on the device from given uniform numbers.  No counterpart in the reference, whose ``generate`` runs one batch of equal
lengths (complexity_deep/models/modeling.py:221-296)."""
from __future__ import annotations

from typing import List, Optional, Sequence, Tuple

import torch

from .. import ops
from ..core.token_routed_mlp import ROUTING_CACHE


class PagedDecoder:
    """CUDA-graph replay of one decode step of all slots of a PagedKVCache, sampling included: attention over every sequence's own
    rows, logits, next token by the slot's rules, which the following step takes up without the host in between.

        dec = PagedDecoder(model, slots=32, pages=1024, page=64, max_rows=4096, keep=2048, recent=256)
        slot, first = dec.add(prompt_ids, uniform=0.3, temperature=0.8, top_k=50, top_p=0.9)
        ids, probs = dec.step(torch.rand(32, device="cuda"))     # [slots] each, overwritten by the next step
        dec.release(slot)

    keep: a sequence is cut back to that many rows when it has `cut` rows (max_rows unless given; keep 0: a sequence with max_rows
    raises).  Which rows stay goes by the attention that steps have paid them, and a prompt's rows come without any: one of more
    than `keep` tokens is first cut when it has cut - keep more, as far as max_rows goes; one of max_rows tokens is cut before its first
    step, to its first rows and the `recent` newest.  Entries of slots that are not in use mean nothing."""

    def __init__(self, model, slots: int, pages: int, page: int = 64, max_rows: int = 2048, max_positions: Optional[int] = None,
                 keep: int = 0, recent: int = 0, warmup: int = 2, cut: Optional[int] = None) -> None:
        if keep and not (0 <= recent <= keep < max_rows):
            raise ValueError("expected 0 <= recent <= keep < max_rows")
        if cut is not None and not 0 < keep < cut <= max_rows:
            raise ValueError("expected 0 < keep < cut <= max_rows")
        device = next(model.parameters()).device
        if device.type != "cuda":
            raise RuntimeError("PagedDecoder needs the model on a CUDA device")
        self.model, self.keep, self.recent, self.cut = model, keep, recent, cut or max_rows
        self._limit = [self.cut] * slots      # rows at which a slot's sequence is cut
        self.cache = model.make_paged_cache(slots, pages, page, max_rows, max_positions, statistics=keep > 0)
        on = dict(device=device)
        self.ids = torch.zeros(slots, 1, dtype=torch.int64, **on)
        self.uniform = torch.zeros(slots, **on)
        self.temperature, self.top_k = torch.zeros(slots, **on), torch.zeros(slots, dtype=torch.int32, **on)
        self.top_p, self.min_p = torch.ones(slots, **on), torch.zeros(slots, **on)
        stream = torch.cuda.Stream(device=device)
        stream.wait_stream(torch.cuda.current_stream(device))
        with torch.no_grad(), torch.cuda.stream(stream):
            for _ in range(warmup):       # builds the packed weights, sets kernel attributes; no slot is in use
                self._eager_step()
        torch.cuda.current_stream(device).wait_stream(stream)
        torch.cuda.synchronize(device)
        self.ids.zero_()                  # fresh version: the capture must contain the dispatch
        ROUTING_CACHE.clear()
        self.graph = torch.cuda.CUDAGraph()
        with torch.no_grad(), torch.cuda.graph(self.graph):
            self.probs = self._eager_step()
        ROUTING_CACHE.clear()             # its entries point into the graph's private pool

    def _eager_step(self) -> torch.Tensor:
        logits = self.model(self.ids, past_key_values=self.cache.as_past(), use_cache=True).logits
        ids, probs = ops.sample_tokens(logits[:, -1], self.uniform, self.temperature, self.top_k, self.top_p, self.min_p)
        self.ids.copy_(ids[:, None])
        self.cache.advance_device()
        return probs

    def add(self, prompt_ids: torch.Tensor, uniform: float = 0.0, temperature: float = 1.0, top_k: int = 50, top_p: float = 0.9,
            min_p: float = 0.0) -> Tuple[int, torch.Tensor]:
        """Runs a prompt [P] and gives it a slot; its rules hold until ``release``.  Returns the slot and the first token drawn
        behind the prompt [1], by `uniform` (0 <= uniform < 1).  A prompt without a slot, rows or pages for it and rules that are no
        numbers are refused before the prompt runs."""
        self.cache.room_for(prompt_ids.numel())
        rules = [(self.temperature, float(temperature)), (self.top_k, max(0, min(int(top_k), 2 ** 31 - 1))), (self.top_p, float(top_p)),
                 (self.min_p, float(min_p)), (self.uniform, float(uniform))]
        with torch.no_grad():
            out = self.model(prompt_ids.view(1, -1).to(self.ids.device), use_cache=True)
        slot = self.cache.add(out.past_key_values)
        self._limit[slot] = min(self.cache.max_rows, max(self.keep, prompt_ids.numel()) + self.cut - self.keep)
        for rule, value in rules:
            rule[slot] = value
        one = slice(slot, slot + 1)
        first, _ = ops.sample_tokens(out.logits[:, -1], self.uniform[one], self.temperature[one], self.top_k[one], self.top_p[one],
                                     self.min_p[one])
        self.ids[slot] = first
        return slot, first

    def step(self, uniform: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
        """The next token of every sequence in use: (ids [slots], their probabilities [slots]), from uniform numbers [slots]."""
        due = [slot for slot, limit in enumerate(self._limit) if self.cache.length(slot) >= limit] if self.keep else []
        if due:
            self.cache.evict(self.keep, self.recent, due)
            for slot in due:
                self._limit[slot] = self.cut
        self.cache.reserve()
        self.uniform.copy_(uniform, non_blocking=True)
        self.graph.replay()
        self.cache.advance_host()
        return self.ids[:, 0], self.probs

    def release(self, slot: int) -> None:
        self.cache.release(slot)


def paged_generate(model, prompts: Sequence[torch.Tensor], max_new_tokens: int = 100, temperature: float = 1.0, top_k: int = 50,
                   top_p: float = 0.9, min_p: float = 0.0, eos_token_id: Optional[int] = None, page: int = 64, keep: int = 0,
                   recent: int = 0, seed: Optional[int] = None) -> List[List[int]]:
    """Continues prompts of any lengths side by side; each stops at the end token (the config's, unless given) or after
    `max_new_tokens`.  temperature 0: greedy.  keep: a sequence is cut back to that many rows whenever it has an eighth (at least a
    page) more, one with a longer prompt for the first time when it has as many more than the prompt.  Returns prompt and
    continuation of each."""
    if not prompts or min(len(p) for p in prompts) < 1:
        raise ValueError("paged_generate needs prompts of at least one token")
    if max_new_tokens < 1:
        return [list(map(int, p)) for p in prompts]
    eos = getattr(model.config, "eos_token_id", None) if eos_token_id is None else eos_token_id
    device = next(model.parameters()).device
    last = max(len(p) for p in prompts) + max_new_tokens
    more = max(page, keep // 8)
    rows = [len(p) + max_new_tokens for p in prompts]       # of each at most
    if keep:
        rows = [min(n, max(keep, len(p)) + more) for n, p in zip(rows, prompts)]
    max_rows = max(rows)
    if keep >= max_rows:
        keep = 0
    dec = PagedDecoder(model, len(prompts), sum(-(-n // page) for n in rows), page, max_rows, last, keep, recent,
                       cut=min(max_rows, keep + more) if keep else None)
    g = torch.Generator(device=device)
    if seed is not None:
        g.manual_seed(seed)
    else:
        g.seed()
    out, slots = [list(map(int, p)) for p in prompts], {}
    first = torch.rand(len(prompts), generator=g, device=device).tolist()
    for i, p in enumerate(prompts):
        slot, token = dec.add(torch.as_tensor(p), first[i], temperature, top_k, top_p, min_p)
        slots[slot] = i
        out[i].append(int(token))
    live = {slot for slot, i in slots.items() if out[i][-1] != eos}
    for slot in slots.keys() - live:
        dec.release(slot)
    for _ in range(max_new_tokens - 1):
        if not live:
            break
        ids, _ = dec.step(torch.rand(len(prompts), generator=g, device=device))
        tokens = ids.tolist()
        for slot in sorted(live):
            out[slots[slot]].append(tokens[slot])
            if tokens[slot] == eos:
                live.discard(slot)
                dec.release(slot)
    return out
