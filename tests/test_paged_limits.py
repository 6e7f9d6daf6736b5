"""What stops a step names the slots that stop it, changes nothing, and is over when they are released or cut back."""
import pytest
import torch

from complexity_deep_b200.core import paged


def _cache(lengths, **kw):
    d = dict(pages=20, page=16, max_rows=48, max_positions=60, device="cpu", statistics=True)
    cache = paged.PagedKVCache(1, len(lengths), 1, 8, **{**d, **kw})
    for n in lengths:
        cache.add([tuple(torch.ones(1, 1, n, 8, dtype=torch.bfloat16) for _ in range(2))])
    return cache


def _steps(cache, n):
    for _ in range(n):
        cache.reserve()
        cache.advance()


@pytest.mark.parametrize("lengths,kw,steps,slots", [([10, 48, 3, 48], {}, 0, [1, 3]), ([10, 40, 3], dict(max_positions=45), 5, [1]),
                                                    ([16, 30, 32, 16], dict(pages=7), 0, [0, 2, 3])])
def test_slots_are_named(lengths, kw, steps, slots):
    cache = _cache(lengths, **kw)
    _steps(cache, steps)
    state = lambda: (cache.free_pages, cache.lengths.tolist(), cache.table.tolist(), cache._table.tolist())  # noqa: E731
    before = state()
    with pytest.raises(RuntimeError) as e:
        cache.reserve()
    assert str(slots) in str(e.value) and state() == before
    for slot in slots:
        cache.release(slot)
    _steps(cache, 1)


def test_cut_back(monkeypatch):
    monkeypatch.setattr(paged.ops, "evict_rows_", lambda *a: None)
    cache = _cache([48, 20])
    with pytest.raises(RuntimeError, match=r"rows: slots \[0\]"):
        cache.reserve()
    cache.evict(30, 4, [0])
    _steps(cache, 10)


def test_slots_of_a_cut(monkeypatch):
    """Any iterable of slots, none and one twice; one that there is not changes nothing."""
    calls = []
    monkeypatch.setattr(paged.ops, "evict_rows_", lambda *a: calls.append(a[3].tolist()))
    cache = _cache([40, 41, 42])
    cache.evict(20, 4, [])
    with pytest.raises(IndexError):
        cache.evict(20, 4, [0, 3])
    assert not calls and cache.lengths.tolist() == [40, 41, 42]
    cache.evict(20, 4, (slot for slot in (2, 0)))
    assert calls == [[40, -1, 42]] and cache.lengths.tolist() == [20, 41, 20] == [cache.length(i) for i in range(3)]
    cache.evict(20, 4, [1, 1])
    assert cache.lengths.tolist() == [20, 20, 20] and cache.free_pages == 20 - 6
