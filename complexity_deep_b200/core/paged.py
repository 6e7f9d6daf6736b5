"""KV cache in pages: the rows of a sequence lie in pages of a pool that a table names, so sequences of different lengths come, grow and
go without a buffer of the largest size for each.  Not part of the reference's API (its cache is a list of tensors that
grow by ``torch.cat``, complexity_deep/core/attention.py:158-161).

``StaticKVCache`` (core.attention) holds a batch of one common length; here every slot has a length and a position of its own, both in
device memory, so a decode step's launches are the same at all lengths (a CUDA graph can hold them).  With ``statistics`` every cached row
has the attention weight that decode steps have given it so far and the position of its token; ``evict`` cuts long sequences
back by them.
"""
from __future__ import annotations

from typing import List, Optional, Sequence

import torch

from .. import ops


class PagedKVCache:
    """`slots` sequences of at most `max_rows` cached rows each, in `pages` pages of `page` rows (of every layer).

    ``add`` takes over a prompt's cache into a free slot, ``reserve`` sees to it that the next step has a place in every sequence in
    use, ``advance`` follows a step, ``evict`` cuts back, ``release`` frees.  A decode step is ``model(ids, past_key_values=cache.as_past(),
    use_cache=True)`` with one id per slot; slots that are not in use take part with any id and give zeros for attention."""

    def __init__(self, num_layers: int, slots: int, kv_heads: int, head_dim: int, pages: int, page: int, max_rows: int,
                 max_positions: int, device, statistics: bool = False) -> None:
        if min(num_layers, slots, pages, page, max_rows, max_positions) < 1:
            raise ValueError("a PagedKVCache needs at least one layer, slot, page, row and position")
        if page not in (16, 32, 64, 128, 256):
            raise ValueError("pages have 16, 32, 64, 128 or 256 rows")
        self.slots, self.pages, self.page = slots, pages, page
        self.max_rows, self.max_positions = max_rows, max_positions
        self.width = -(-max_rows // page)
        shape = (num_layers, pages, kv_heads, page, head_dim)
        self.k = torch.zeros(shape, dtype=torch.bfloat16, device=device)
        self.v = torch.zeros_like(self.k)
        # what a step reads on the device; entries of the table without a page lie outside the pool
        self.table = torch.full((slots, self.width), pages, dtype=torch.int32, device=device)
        self.lengths = torch.full((slots,), -1, dtype=torch.int32, device=device)
        self.positions = torch.zeros(slots, dtype=torch.int32, device=device)
        self.live = torch.zeros(slots, dtype=torch.int32, device=device)
        rows = (num_layers, slots, kv_heads, self.width * page)
        self.weights = torch.zeros(rows, dtype=torch.float32, device=device) if statistics else None
        self.row_positions = torch.zeros(rows, dtype=torch.int32, device=device) if statistics else None
        # and on the host
        self._length: List[int] = [-1] * slots
        self._position: List[int] = [0] * slots
        self._pages: List[List[int]] = [[] for _ in range(slots)]
        self._free = list(range(pages - 1, -1, -1))
        self._table = torch.full((slots, self.width), pages, dtype=torch.int32)
        self.layers = [PagedKVLayer(self, i) for i in range(num_layers)]

    # ------------------------------------------------------------------ host side
    def length(self, slot: int) -> int:
        """Cached rows of the slot, -1 if it is not in use."""
        return self._length[slot]

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def as_past(self) -> list:
        """What a forward call takes as ``past_key_values``."""
        return self.layers

    def _take(self, slot: int, count: int) -> None:
        """`count` more pages for the slot (of the host's table; ``_send`` brings it to the device)."""
        if count > len(self._free):
            raise RuntimeError(f"no page left: {count} wanted, {len(self._free)} of {self.pages} free")
        for _ in range(count):
            self._table[slot, len(self._pages[slot])] = self._free[-1]
            self._pages[slot].append(self._free.pop())

    def _give_back(self, slot: int, count: int) -> None:
        """Keeps the slot's first `count` pages."""
        self._table[slot, count:] = self.pages
        self._free.extend(reversed(self._pages[slot][count:]))
        del self._pages[slot][count:]

    def _send(self) -> None:
        self.table.copy_(self._table, non_blocking=True)     # from pageable memory: the host's copy is free when the call returns

    def room_for(self, rows: int) -> int:
        """The slot that a prompt of so many tokens gets; raises if there is no slot, row or page for it."""
        if -1 not in self._length:
            raise RuntimeError(f"all {self.slots} slots are in use")
        if not 1 <= rows <= self.max_rows or rows > self.max_positions:
            raise ValueError(f"{rows} tokens do not fit sequences of {self.max_rows} rows")
        count = -(-rows // self.page)
        if count > len(self._free):
            raise RuntimeError(f"no page left: {count} wanted, {len(self._free)} of {self.pages} free")
        return self._length.index(-1)

    def add(self, past_key_values, row: int = 0) -> int:
        """Takes over the cache of sequence `row` of a prompt (list of (k, v) [B, kv heads, P, D]) and returns the slot.  What does not
        fit is refused before anything is changed."""
        layers, _, kv_heads, _, dim = self.k.shape
        B, _, rows, _ = shape = past_key_values[0][0].shape
        if len(past_key_values) != layers or not -B <= row < B or any(t.shape != (B, kv_heads, rows, dim) for p in past_key_values for t in p):
            raise ValueError(f"expected sequence {row} of {layers} layers of [B, {kv_heads}, rows, {dim}], the first of "
                             f"{len(past_key_values)} is {list(shape)}")
        slot = self.room_for(rows)
        count = -(-rows // self.page)
        self._take(slot, count)
        try:
            ids = torch.tensor(self._pages[slot], device=self.k.device)
            for i, pair in enumerate(past_key_values):
                for pool, t in zip((self.k, self.v), pair):
                    t = torch.nn.functional.pad(t[row], (0, 0, 0, count * self.page - rows))
                    pool[i, ids] = t.unflatten(1, (count, self.page)).transpose(0, 1)
            if self.weights is not None:
                self.weights[:, slot, :, :rows] = 0.0
                self.row_positions[:, slot, :, :rows] = torch.arange(rows, dtype=torch.int32, device=self.k.device)
        except BaseException:                             # no memory for the copies
            self._give_back(slot, 0)
            raise
        self._length[slot] = self._position[slot] = rows
        self.lengths[slot] = self.positions[slot] = rows
        self.live[slot] = 1
        self._send()
        return slot

    def release(self, slot: int) -> None:
        if self._length[slot] < 0:
            raise ValueError(f"slot {slot} is not in use")
        self._give_back(slot, 0)
        self._length[slot] = -1
        self.lengths[slot] = -1
        self.live[slot] = 0
        self._send()

    def full(self) -> bool:
        """Whether a sequence has no row left for the next step."""
        return any(n >= self.max_rows for n in self._length)

    def reserve(self) -> None:
        """A place for the next token in every sequence in use.  Raises before anything is changed if one has none, and names those
        slots: without them (``release``), or with fewer rows in them (``evict``), the others go on."""
        full = [slot for slot, n in enumerate(self._length) if n >= self.max_rows]
        if full:
            raise RuntimeError(f"a sequence has all of its {self.max_rows} rows: slots {full}")
        last = [slot for slot, (n, p) in enumerate(zip(self._length, self._position)) if n >= 0 and p >= self.max_positions]
        if last:
            raise RuntimeError(f"a sequence is at the last of {self.max_positions} positions: slots {last}")
        wanting = [slot for slot, n in enumerate(self._length) if n >= 0 and n == len(self._pages[slot]) * self.page]
        if len(wanting) > len(self._free):
            raise RuntimeError(f"no page left: {len(wanting)} wanted, {len(self._free)} of {self.pages} free: slots {wanting}")
        for slot in wanting:
            self._take(slot, 1)
        if wanting:
            self._send()

    # ------------------------------------------------------------------ steps
    def advance_device(self) -> None:
        """Moves lengths and positions of the slots in use by one token (stream ordered, capturable)."""
        self.lengths.add_(self.live)
        self.positions.add_(self.live)

    def advance_host(self) -> None:
        for slot, n in enumerate(self._length):
            if n >= 0:
                self._length[slot] = n + 1
                self._position[slot] += 1

    def advance(self) -> None:
        self.advance_device()
        self.advance_host()

    def evict(self, keep: int, recent: int, slots: Optional[Sequence[int]] = None) -> None:
        """Cuts every sequence (of those slots, where they are given) of more than `keep` rows back to `keep` per layer and KV head: the
        last `recent` tokens and the rows of largest weight (``ops.evict_rows_``).  The pages behind them are free afterwards.  Weights
        are those of the steps so far: a prompt's rows come with none."""
        if self.weights is None:
            raise RuntimeError("evict needs a cache with statistics")
        keep, recent = (min(n, self.width * self.page) for n in (keep, recent))
        lengths = self.lengths
        chosen = list(range(self.slots) if slots is None else slots)
        if not chosen:
            return
        if slots is not None:                             # the others look as if they were not in use
            these = torch.zeros(self.slots, dtype=torch.bool)
            these[chosen] = True
            these = these.to(lengths.device)
            lengths = torch.where(these, lengths, -1)
        ops.evict_rows_(self.k, self.v, self.table, lengths, self.positions, self.weights, self.row_positions, keep, recent)
        if slots is None:
            self.lengths.clamp_(max=keep)
        else:
            self.lengths.copy_(torch.where(these, self.lengths.clamp(max=keep), self.lengths))
        for slot in chosen:
            if self._length[slot] > keep:
                self._length[slot] = keep
                self._give_back(slot, -(-keep // self.page))
        self._send()


class PagedKVLayer:
    """One layer's part of a PagedKVCache, passed as that layer's ``past_key_value``."""

    def __init__(self, cache: PagedKVCache, index: int) -> None:
        self.cache, self.index = cache, index

    def step(self, qkv, q_w, k_w, cos, sin, eps, hq, hkv, head_dim) -> torch.Tensor:
        """Attention of one new token per slot, which is stored on the way (``ops.paged_step_attention``)."""
        c, i = self.cache, self.index
        return ops.paged_step_attention(qkv, q_w, k_w, cos, sin, eps, hq, hkv, head_dim, c.k[i], c.v[i], c.table, c.lengths,
                                        c.positions, weights=None if c.weights is None else c.weights[i],
                                        row_positions=None if c.row_positions is None else c.row_positions[i])
