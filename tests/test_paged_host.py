"""What the operators on a paged cache and the sampling refuse, through the C interface (argument checks come before any CUDA call)
and through the tensor wrappers (no CPU path)."""
import ctypes

import pytest
import torch

from complexity_deep_b200 import _lib, ops

A = 4096                                  # an aligned address that nobody follows
INVALID, UNSUPPORTED = 1, 3


def _cache(**kw):
    d = dict(k=A, v=A, stride_p=4096, stride_h=1024, stride_t=64, table=A, table_stride=4, lengths=A, weights=None, pages=8,
             page=16, width=4)
    d.update(kw)
    return _lib.Paged(**d)


def _attend(c, q=A, stride=256, B=2, hq=4, hkv=2, D=64, out=A, ws=None, n=0):
    return _lib.load().cd_paged_attention(None if c is None else ctypes.byref(c), q, stride, 0.125, B, hq, hkv, D, out, ws, n, None)


@pytest.mark.parametrize("change,status", [
    (dict(k=None), INVALID), (dict(v=None), INVALID), (dict(table=None), INVALID), (dict(lengths=None), INVALID),
    (dict(k=A + 8), INVALID), (dict(v=A + 2), INVALID), (dict(stride_p=4100), INVALID), (dict(stride_h=4), INVALID),
    (dict(stride_t=63), INVALID), (dict(stride_t=-64), INVALID), (dict(pages=0), INVALID), (dict(page=0), INVALID),
    (dict(width=0), INVALID), (dict(table_stride=-1), INVALID), (dict(page=24), UNSUPPORTED), (dict(page=512), UNSUPPORTED),
    (dict(page=256, width=1 << 23), UNSUPPORTED)])
def test_cache_arguments(change, status):
    assert _attend(_cache(**change)) == status


@pytest.mark.parametrize("change,status", [
    (dict(q=None), INVALID), (dict(out=None), INVALID), (dict(q=A + 2), INVALID), (dict(stride=129), INVALID), (dict(B=0), INVALID),
    (dict(hq=5), INVALID), (dict(hkv=0), INVALID), (dict(D=80), UNSUPPORTED), (dict(hq=34), UNSUPPORTED), (dict(D=63), INVALID)])
def test_attention_arguments(change, status):
    assert _attend(_cache(), **change) == status
    assert _attend(None) == INVALID


def test_workspaces():
    lib = _lib.load()
    n = lib.cd_paged_attention_workspace_bytes(2, 4, 2, 64, 16, 4, 1)
    assert n >= 2 * 4 * 64 * 4
    assert _attend(_cache(weights=A)) == INVALID and _attend(_cache(weights=A), ws=A, n=n - 1) == INVALID
    assert _attend(_cache(weights=A), ws=A + 4, n=n) == INVALID and _attend(_cache(weights=A + 4), ws=A, n=n) == INVALID
    assert lib.cd_paged_attention_workspace_bytes(2, 4, 2, 96, 16, 4, 1) == 0
    assert lib.cd_evict_rows_workspace_bytes(1, 2, 2, 16, 4, 0) == 0


def test_step_arguments():
    lib = _lib.load()
    good = dict(q_w=A, k_w=A, cos_t=A, sin_t=A, positions=A, row_positions=None, eps=1e-6, table_rows=64)
    for change in (dict(cos_t=None), dict(sin_t=None), dict(positions=None), dict(table_rows=0), dict(q_w=None), dict(k_w=None)):
        step = _lib.PagedStep(**{**good, **change})
        assert lib.cd_paged_step_attention(ctypes.byref(_cache()), ctypes.byref(step), A, 0.125, 2, 4, 2, 64, A, None, 0, None) == INVALID
    assert lib.cd_paged_step_attention(ctypes.byref(_cache()), None, A, 0.125, 2, 4, 2, 64, A, None, 0, None) == INVALID


def test_evict_arguments():
    lib = _lib.load()
    good = dict(positions=A, row_positions=A, weights_out=A, row_positions_out=A, keep=8, recent=2)
    n = lib.cd_evict_rows_workspace_bytes(1, 2, 2, 16, 4, 8)

    def call(c, layers=1, stride=0, ws=A, size=n, **change):
        e = _lib.Evict(**{**good, **change})
        return lib.cd_evict_rows(ctypes.byref(c), ctypes.byref(e), layers, stride, 2, 2, 64, ws, size, None)

    for change in (dict(positions=None), dict(row_positions=None), dict(weights_out=None), dict(row_positions_out=None), dict(keep=0),
                   dict(recent=-1), dict(recent=9), dict(layers=0), dict(stride=12), dict(weights_out=2 * A)):
        assert call(_cache(weights=A), **change) == INVALID
    assert call(_cache()) == INVALID
    if n:
        assert call(_cache(weights=A), ws=None) == INVALID and call(_cache(weights=A), size=n - 1) == INVALID


def test_sample_arguments():
    lib = _lib.load()

    def call(logits=A, ld=100, B=2, V=100, uniform=A, ids=A, probs=A):
        r = _lib.Sample(uniform=uniform, temperature=1.0, top_p=1.0)
        return lib.cd_sample_tokens(logits, 0, ld, B, V, ctypes.byref(r), ids, probs, None)

    for change in (dict(logits=None), dict(uniform=None), dict(ids=None), dict(probs=None), dict(B=0), dict(V=0), dict(ld=-1)):
        assert call(**change) == INVALID
    assert call(V=(1 << 18) + 1, ld=1 << 19) == UNSUPPORTED
    assert lib.cd_sample_tokens(A, 0, 100, 2, 100, None, A, A, None) == INVALID


def test_wrappers_have_no_cpu_path():
    pool, table, n = torch.zeros(4, 2, 16, 64, dtype=torch.bfloat16), torch.zeros(1, 2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    qkv, cos = torch.zeros(1, 8 * 64, dtype=torch.bfloat16), torch.zeros(40, 64)
    stat, pos = torch.zeros(1, 2, 32), torch.zeros(1, 2, 32, dtype=torch.int32)
    with pytest.raises(RuntimeError):
        ops.paged_attention(qkv, pool, pool, table, n, 4, 2, 64)
    with pytest.raises(RuntimeError):
        ops.paged_step_attention(qkv, None, None, cos, cos, 1e-6, 4, 2, 64, pool, pool, table, n, n)
    with pytest.raises(RuntimeError):
        ops.evict_rows_(pool, pool, table, n, n, stat, pos, 8, 2)
    with pytest.raises(RuntimeError):
        ops.sample_tokens(torch.zeros(1, 10), torch.zeros(1))


# --------------------------------------------------------------------------- bookkeeping of the cache
def _prompt(rows, layers=2, hkv=2, dim=8):
    g = torch.Generator().manual_seed(rows)
    return [tuple(torch.randn(1, hkv, rows, dim, generator=g).to(torch.bfloat16) for _ in range(2)) for _ in range(layers)]


def _held(cache, slot, n):
    ids = cache.table[slot, : -(-n // cache.page)].long()
    return cache.k[:, ids].transpose(1, 2).flatten(2, 3)[:, :, :n]


def test_cache_takes_over_grows_and_frees():
    from complexity_deep_b200.core.paged import PagedKVCache
    cache = PagedKVCache(2, 3, 2, 8, pages=6, page=16, max_rows=48, max_positions=60, device="cpu", statistics=True)
    a, b = _prompt(16), _prompt(20)
    cache.weights.fill_(9.0)
    s0, s1 = cache.add(a), cache.add(b)
    assert (s0, s1, cache.free_pages) == (0, 1, 3) and cache.lengths.tolist() == [16, 20, -1] == [cache.length(i) for i in range(3)]
    assert torch.equal(_held(cache, 0, 16), torch.stack([p[0][0] for p in a])) and torch.equal(_held(cache, 1, 20), torch.stack([p[0][0] for p in b]))
    assert bool((cache.weights[:, 1, :, :20] == 0).all()) and bool((cache.weights[:, 1, :, 20:] == 9).all())
    assert cache.row_positions[0, 1, 0, :20].tolist() == list(range(20))
    cache.reserve()                                           # slot 0 has filled its page, slot 1 has room
    assert cache.free_pages == 2 and int(cache.table[0, 1]) < 6 and int(cache.table[0, 2]) == 6
    for _ in range(12):
        cache.reserve()
        cache.advance()
    assert cache.lengths.tolist() == [28, 32, -1] and cache.positions.tolist() == [28, 32, 0]
    cache.reserve()
    assert cache.free_pages == 1 and len(set(cache.table[cache.table < 6].tolist())) == 5
    cache.release(0)
    assert cache.free_pages == 3 and cache.lengths.tolist() == [-1, 32, -1] and cache.table[0].tolist() == [6, 6, 6]
    cache.advance()
    assert cache.lengths.tolist() == [-1, 33, -1]             # slots that are not in use stay as they are
    assert cache.add(_prompt(40)) == 0 and cache.free_pages == 0
    with pytest.raises(RuntimeError):
        cache.add(_prompt(3))
    with pytest.raises(ValueError):
        cache.release(2)


def test_cache_limits():
    from complexity_deep_b200.core.paged import PagedKVCache
    with pytest.raises(ValueError):
        PagedKVCache(1, 1, 1, 8, pages=1, page=24, max_rows=8, max_positions=8, device="cpu")
    cache = PagedKVCache(2, 1, 2, 8, pages=3, page=16, max_rows=20, max_positions=40, device="cpu")
    with pytest.raises(ValueError):
        cache.add(_prompt(21))
    cache.add(_prompt(19))
    cache.reserve()
    cache.advance()
    assert cache.full()
    with pytest.raises(RuntimeError, match="rows"):
        cache.reserve()
    with pytest.raises(RuntimeError, match="statistics"):
        cache.evict(8, 2)


def test_cache_bookkeeping_of_an_eviction(monkeypatch):
    from complexity_deep_b200.core import paged
    cache = paged.PagedKVCache(2, 2, 2, 8, pages=8, page=16, max_rows=64, max_positions=64, device="cpu", statistics=True)
    cache.add(_prompt(60))
    cache.add(_prompt(18))
    calls = []
    monkeypatch.setattr(paged.ops, "evict_rows_", lambda *a: calls.append(a[-2:]))
    cache.evict(20, 4)
    assert calls == [(20, 4)] and cache.lengths.tolist() == [20, 18] == [cache.length(0), cache.length(1)] and cache.free_pages == 4
    assert int(cache.table[0, 1]) < 8 and cache.table[0, 2:].tolist() == [8, 8] and cache.positions.tolist() == [60, 18]


def test_command_line_prompts():
    from complexity_deep_b200 import cli
    assert cli.parse_prompts(["1,2", "3"], equal=False) == [[1, 2], [3]]
    for texts, equal in ((["1,2", "3"], True), (["1", ""], False)):
        with pytest.raises(SystemExit):
            cli.parse_prompts(texts, equal)


def test_generate_without_work():
    from complexity_deep_b200.models import paged_generate
    assert paged_generate(None, [[3, 1], torch.tensor([4])], max_new_tokens=0) == [[3, 1], [4]]
    for prompts in ([], [[3], []]):
        with pytest.raises(ValueError, match="at least one token"):
            paged_generate(None, prompts)
