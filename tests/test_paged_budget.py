"""When a decoder cuts its sequences back (on the CPU, without the kernels): each at its own number of rows, a long prompt only
when steps have paid its rows attention, and never more pages than were counted ahead."""
import types

import pytest
import torch

from complexity_deep_b200.core import paged
from complexity_deep_b200.models import PagedDecoder, serving


class _Decoder(PagedDecoder):
    """A decoder whose steps compute nothing."""

    def __init__(self, model, slots, pages, page, max_rows, max_positions=None, keep=0, recent=0, warmup=2, cut=None):
        if cut is not None and not 0 < keep < cut <= max_rows:
            raise ValueError
        self.cache = paged.PagedKVCache(1, slots, 1, 8, pages, page, max_rows, max_positions or max_rows, "cpu", keep > 0)
        self.model, self.keep, self.recent, self.cut = model, keep, recent, cut or max_rows
        self._limit = [self.cut] * slots
        self.ids, self.uniform = torch.zeros(slots, 1, dtype=torch.int64), torch.zeros(slots)
        self.temperature, self.top_k = torch.zeros(slots), torch.zeros(slots, dtype=torch.int32)
        self.top_p, self.min_p, self.probs = torch.ones(slots), torch.zeros(slots), torch.zeros(slots)
        self.graph = types.SimpleNamespace(replay=self.cache.advance_device)
        made.append(self)

    def step(self, uniform):
        out = super().step(uniform)
        self.seen.append([self.cache.length(i) for i in range(self.cache.slots)])
        assert self.cache.lengths.tolist() == self.seen[-1]
        assert self.cache.free_pages == self.cache.pages - sum(len(p) for p in self.cache._pages)
        return out

    seen, cuts = [], []


made = []


def _model(ids, use_cache):
    n = ids.shape[1]
    return types.SimpleNamespace(past_key_values=[tuple(torch.zeros(1, 1, n, 8, dtype=torch.bfloat16) for _ in range(2))],
                                 logits=torch.zeros(1, n, 11))


@pytest.fixture
def decoder(monkeypatch):
    made.clear()
    monkeypatch.setattr(_Decoder, "seen", [])
    monkeypatch.setattr(_Decoder, "cuts", [])

    def evict(k, v, table, lengths, positions, weights, row_positions, keep, recent):
        _Decoder.cuts.append([(i, int(n)) for i, n in enumerate(lengths) if n > keep])
    monkeypatch.setattr(paged.ops, "evict_rows_", evict)
    monkeypatch.setattr(serving.ops, "sample_tokens", lambda x, u, *rules: (torch.zeros(1, dtype=torch.int64), u))
    return _Decoder


def _run(dec, steps):
    for _ in range(steps):
        dec.step(torch.zeros(dec.cache.slots))
    return dec.seen


def test_each_sequence_at_its_own_limit(decoder):
    dec = decoder(_model, 3, 40, 16, 120, 400, keep=48, recent=8, cut=64)
    for n in (10, 60, 90):
        dec.add(torch.arange(n))
    seen = _run(dec, 100)
    # 10 tokens: at 64 rows; 60 and 90: when 16 steps have seen the whole prompt, at 64 from then on
    first = [next(i for i, c in enumerate(dec.cuts) if any(s == slot for s, _ in c)) for slot in range(3)]
    assert [dict(dec.cuts[f])[slot] for slot, f in enumerate(first)] == [64, 76, 106]
    assert all(n == 64 for slot in range(3) for c in dec.cuts[first[slot] + 1:] for s, n in c if s == slot)
    assert max(max(x) for x in seen) == 106 and [max(x[slot] for x in seen[40:]) for slot in range(3)] == [64, 64, 64]
    assert dec.cache.positions.tolist() == [110, 160, 190]


def test_without_a_cut_of_its_own(decoder):
    """max_rows is the limit, and of that sequence alone: one that has just come keeps its prompt."""
    dec = decoder(_model, 2, 40, 16, 80, 400, keep=32, recent=8)
    dec.add(torch.arange(70))
    _run(dec, 8)
    dec.add(torch.arange(60))
    seen = _run(dec, 4)
    assert [list(c) for c in dec.cuts] == [[(0, 80)]] and seen[-1] == [34, 64]
    full = decoder(_model, 1, 5, 16, 80, 400, keep=32, recent=8)
    full.add(torch.arange(80))                               # no room for a step: cut at once
    full.step(torch.zeros(1))
    assert full.cuts[-1] == [(0, 80)] and full.cache.length(0) == 33


def test_a_slot_that_is_given_back(decoder):
    dec = decoder(_model, 1, 10, 16, 120, 400, keep=32, recent=8, cut=48)
    slot, _ = dec.add(torch.arange(100))
    _run(dec, 3)
    dec.release(slot)
    dec.add(torch.arange(10))
    _run(dec, 80)
    assert dec.cuts and all(n == 48 for c in dec.cuts for _, n in c)
    with pytest.raises(ValueError):
        decoder(_model, 1, 10, 16, 120, keep=48, cut=48)


@pytest.mark.parametrize("keep", [100, 24])
def test_paged_generate_stays_within_its_budget(decoder, monkeypatch, keep):
    monkeypatch.setattr(serving, "PagedDecoder", decoder)
    monkeypatch.setattr(torch, "Generator", lambda device: types.SimpleNamespace(manual_seed=lambda s: None, seed=lambda: None))
    monkeypatch.setattr(torch, "rand", lambda n, generator, device: torch.zeros(n))
    model = types.SimpleNamespace(config=types.SimpleNamespace(eos_token_id=None), parameters=lambda: iter([torch.zeros(1)]))
    monkeypatch.setattr(decoder, "model", None, raising=False)
    real = decoder.add
    monkeypatch.setattr(decoder, "add", lambda self, p, *a: (setattr(self, "model", _model), real(self, p, *a))[1])
    prompts = [[1] * n for n in (300, 5, 110)]
    out = serving.paged_generate(model, prompts, 250, page=16, keep=keep, recent=4)
    assert [len(x) for x in out] == [550, 255, 360]
    dec, more = made[0], max(16, keep // 8)
    for slot, p in enumerate(prompts):
        counts = [n for c in dec.cuts for s, n in c if s == slot]
        assert counts[0] == max(keep, len(p)) + more and set(counts[1:]) == {keep + more}
        assert max(x[slot] for x in dec.seen) <= max(keep, len(p)) + more
        # the pages of each, counted ahead
    assert dec.cache.pages == sum(-(-min(len(p) + 250, max(keep, len(p)) + more) // 16) for p in prompts)


def test_paged_generate_with_nothing_to_cut(decoder, monkeypatch):
    monkeypatch.setattr(serving, "PagedDecoder", decoder)
    monkeypatch.setattr(torch, "Generator", lambda device: types.SimpleNamespace(manual_seed=lambda s: None, seed=lambda: None))
    monkeypatch.setattr(torch, "rand", lambda n, generator, device: torch.zeros(n))
    model = types.SimpleNamespace(config=types.SimpleNamespace(eos_token_id=None), parameters=lambda: iter([torch.zeros(1)]))
    real = decoder.add
    monkeypatch.setattr(decoder, "add", lambda self, p, *a: (setattr(self, "model", _model), real(self, p, *a))[1])
    serving.paged_generate(model, [[1] * 30, [2]], 10, page=16, keep=40, recent=4)
    assert not made[0].cuts and made[0].cache.weights is None and made[0].cache.max_rows == 40
    serving.paged_generate(model, [[1] * 30, [2]], 10, page=16, keep=39, recent=4)
    assert not made[1].cuts and made[1].cache.max_rows == 40
