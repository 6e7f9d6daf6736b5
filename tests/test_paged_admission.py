"""Prompts that a paged cache has no place for, or that are not of its shape, are refused before anything has run or changed."""
import types

import pytest
import torch

from complexity_deep_b200.core.paged import PagedKVCache
from complexity_deep_b200.models import PagedDecoder


def _cache(**kw):
    d = dict(num_layers=2, slots=2, kv_heads=2, head_dim=8, pages=6, page=16, max_rows=48, max_positions=60, device="cpu",
             statistics=True)
    return PagedKVCache(**{**d, **kw})


def _prompt(rows, layers=2, hkv=2, dim=8, batch=1):
    return [tuple(torch.ones(batch, hkv, rows, dim, dtype=torch.bfloat16) for _ in range(2)) for _ in range(layers)]


def _state(cache):
    return (cache.free_pages, [cache.length(i) for i in range(cache.slots)], cache.lengths.tolist(), cache.live.tolist(),
            cache.table.tolist(), cache._table.tolist())


@pytest.mark.parametrize("past,row", [(_prompt(20, layers=1), 0), (_prompt(20, layers=3), 0), (_prompt(20, hkv=1), 0), (_prompt(20, hkv=3), 0),
                                      (_prompt(20, dim=16), 0), (_prompt(20)[:1] + _prompt(21)[:1], 0), (_prompt(20), 1), (_prompt(20), -2),
                                      (_prompt(0), 0), (_prompt(49), 0)])
def test_other_shapes(past, row):
    cache = _cache()
    cache.add(_prompt(7, batch=3), 2)
    before = _state(cache)
    with pytest.raises(ValueError):
        cache.add(past, row)
    assert _state(cache) == before


def test_a_copy_that_fails_leaves_no_page_behind(monkeypatch):
    cache = _cache()
    before = _state(cache)

    def out_of_memory(*a):
        raise torch.OutOfMemoryError("made up")
    with monkeypatch.context() as m:
        m.setattr(torch.nn.functional, "pad", out_of_memory)
        with pytest.raises(torch.OutOfMemoryError):
            cache.add(_prompt(20))
    assert _state(cache) == before
    assert cache.add(_prompt(20)) == 0 and cache.free_pages == 4


class _Refused:
    def __call__(self, *a, **k):
        raise AssertionError("the prompt has run")


def _decoder(cache, model):
    dec = object.__new__(PagedDecoder)                       # its constructor captures a step on a GPU
    dec.model, dec.cache, dec.keep, dec.cut, dec._limit = model, cache, 0, cache.max_rows, [cache.max_rows] * cache.slots
    dec.ids, dec.uniform = torch.zeros(cache.slots, 1, dtype=torch.int64), torch.zeros(cache.slots)
    dec.temperature, dec.top_k = torch.zeros(cache.slots), torch.zeros(cache.slots, dtype=torch.int32)
    dec.top_p, dec.min_p = torch.ones(cache.slots), torch.zeros(cache.slots)
    return dec


@pytest.mark.parametrize("tokens,rules,error", [(49, {}, ValueError), (0, {}, ValueError), (5, dict(temperature="hot"), ValueError),
                                                (5, dict(top_k=None), TypeError), (5, dict(uniform=None), TypeError)])
def test_decoder_refuses_ahead_of_the_prompt(tokens, rules, error):
    cache = _cache()
    before = _state(cache)
    with pytest.raises(error):
        _decoder(cache, _Refused()).add(torch.arange(tokens), **rules)
    assert _state(cache) == before


def test_decoder_without_slots_or_pages():
    cache = _cache(pages=4)
    cache.add(_prompt(48))
    with pytest.raises(RuntimeError, match="no page left"):
        _decoder(cache, _Refused()).add(torch.arange(17))
    cache.add(_prompt(3))
    with pytest.raises(RuntimeError, match="slots"):
        _decoder(cache, _Refused()).add(torch.arange(3))


def test_rules_of_any_size(monkeypatch):
    """A top-k beyond 32 bits keeps every token, one below zero too."""
    from complexity_deep_b200.models import serving
    cache = _cache()
    out = types.SimpleNamespace(past_key_values=_prompt(5), logits=torch.zeros(1, 5, 11))
    dec = _decoder(cache, lambda ids, use_cache: out)
    seen = []
    monkeypatch.setattr(serving.ops, "sample_tokens", lambda x, u, t, k, p, m: (seen.append(int(k)), torch.zeros(1, dtype=torch.int64))[::-1])
    for k in (2 ** 40 + 3, -7):
        dec.add(torch.arange(5), top_k=k)
    assert seen == [2 ** 31 - 1, 0]
