"""Cuts of a running decoder: of chosen sequences only, and of a long prompt by the attention that steps have paid its rows."""
import pytest
import torch

import paged_cases as cases

pytestmark = pytest.mark.gpu


def _model(seed=0):
    from complexity_deep_b200.models import ComplexityConfig, ComplexityModel
    torch.manual_seed(seed)
    cfg = ComplexityConfig(vocab_size=500, hidden_size=256, intermediate_size=512, num_hidden_layers=2, num_attention_heads=4,
                           num_key_value_heads=2, num_experts=4, eos_token_id=-1)
    return cfg, ComplexityModel(cfg).to("cuda", torch.bfloat16).eval()


def _same(a, b):
    return torch.equal(a.view(torch.int16), b.view(torch.int16))


def test_chosen_slots():
    from complexity_deep_b200.core.paged import PagedKVCache
    cache = PagedKVCache(2, 3, 2, 64, pages=20, page=16, max_rows=96, max_positions=200, device="cuda", statistics=True)
    g = torch.Generator().manual_seed(1)
    for n in (70, 90, 65):
        cache.add([tuple(torch.randn(1, 2, n, 64, generator=g).to(torch.bfloat16).cuda() for _ in range(2)) for _ in range(2)])
    cache.weights.copy_(torch.rand(cache.weights.shape, generator=g))
    w, pos, k, table = (t.cpu() for t in (cache.weights, cache.row_positions, cache.k, cache.table))
    cache.evict(40, 8, [0, 2])
    assert cache.lengths.tolist() == [40, 90, 40] == [cache.length(i) for i in range(3)] and cache.free_pages == 20 - 3 - 6 - 3
    for layer in range(2):
        assert _same(cases_rows(cache.k[layer].cpu(), table, 1, 90), cases_rows(k[layer], table, 1, 90))
        assert torch.equal(cache.weights[layer, 1].cpu(), w[layer, 1]) and torch.equal(cache.row_positions[layer, 1].cpu(), pos[layer, 1])
        for slot, n in ((0, 70), (2, 65)):
            for h in range(2):
                src = cases.evict(w[layer, slot, h].tolist(), pos[layer, slot, h].tolist(), n, n - 8, 40)
                assert cache.row_positions[layer, slot, h, :40].tolist() == pos[layer, slot, h][src].tolist()
                assert _same(cases_rows(cache.k[layer].cpu(), table, slot, 40)[h], cases_rows(k[layer], table, slot, n)[h][src])


def cases_rows(pool, table, b, n):
    ids = table[b, : -(-n // pool.shape[2])].long()
    return pool[ids].transpose(0, 1).flatten(1, 2)[:, :n].contiguous()


def test_first_cut_of_a_long_prompt(monkeypatch):
    """A prompt of three times the budget: its first cut comes behind a page of steps, and the rows that they have weighed most stay,
    wherever in the prompt they lie."""
    from complexity_deep_b200.core.paged import PagedKVCache
    from complexity_deep_b200.models import PagedDecoder, paged_generate
    cfg, model = _model(2)
    real_evict, real_step, cuts, lengths = PagedKVCache.evict, PagedDecoder.step, [], []

    def evict(self, keep, recent, slots=None):
        w, pos, n = self.weights.cpu(), self.row_positions.cpu(), [self.length(s) for s in range(self.slots)]
        real_evict(self, keep, recent, slots)
        cuts.append((w, pos, n, self.row_positions.cpu()))

    def step(self, uniform):
        out = real_step(self, uniform)
        lengths.append([self.cache.length(s) for s in range(self.cache.slots)])
        assert lengths[-1] == self.cache.lengths.tolist()
        return out
    monkeypatch.setattr(PagedKVCache, "evict", evict)
    monkeypatch.setattr(PagedDecoder, "step", step)
    g = torch.Generator().manual_seed(3)
    prompts = [torch.randint(0, 500, (n,), generator=g) for n in (120, 20)]
    out = paged_generate(model, prompts, 60, 0.9, 50, 0.95, page=16, keep=40, recent=6, seed=4)
    assert [len(x) for x in out] == [180, 80]
    assert [n[0] for n in lengths[:18]] == [121 + i for i in range(16)] + [41, 42] and max(n[1] for n in lengths) == 56
    assert max(n[0] for n in lengths[16:]) == 56
    w, pos, n, after = cuts[0]
    assert n == [136, 36]
    middle = 0
    for layer in range(2):
        for h in range(2):
            mine = w[layer, 0, h, :136]
            assert bool((mine > 0).all()) and abs(float(mine.sum()) - 2 * 16) < 1e-2        # 16 steps, two heads of queries each
            stay = cases.evict(mine.tolist(), pos[layer, 0, h].tolist(), 136, 130, 40)
            assert after[layer, 0, h, :40].tolist() == pos[layer, 0, h][stay].tolist()
            assert int(mine.argmax()) in stay
            middle += sum(40 <= i < 130 for i in stay)
    assert middle > 0                                        # without weights the first rows and the newest would stay
