"""Numbers that no 32 bits hold mean what they say: a budget that no sequence reaches, a top-k of everything."""
import pytest
import torch

import paged_cases as cases

pytestmark = pytest.mark.gpu
LARGE = [2 ** 31 - 1, 2 ** 31, 2 ** 32 + 1, 2 ** 32 + 8, 2 ** 40]


@pytest.mark.parametrize("keep", LARGE)
def test_eviction(keep):
    from complexity_deep_b200 import ops
    from complexity_deep_b200.core.paged import PagedKVCache
    k, v, table = cases.make_cache([40], 1, 64, 16, 1, rest=0.0)
    kd, vd, n = k.cuda(), v.cuda(), torch.tensor([40], dtype=torch.int32, device="cuda")
    w = torch.rand(1, 1, 48, generator=torch.Generator().manual_seed(2))
    pos = torch.arange(48, dtype=torch.int32).flip(0).view(1, 1, 48)
    for recent in (0, 3, keep):
        wd, pd = w.cuda(), pos.cuda()
        ops.evict_rows_(kd, vd, table.cuda(), n, n, wd, pd, keep, recent)
        assert torch.equal(kd.cpu(), k) and torch.equal(vd.cpu(), v) and torch.equal(wd.cpu(), w) and torch.equal(pd.cpu(), pos)
    cache = PagedKVCache(1, 1, 1, 64, pages=3, page=16, max_rows=48, max_positions=60, device="cuda", statistics=True)
    cache.add([(k[table[0].long()].transpose(0, 1).flatten(1, 2)[None, :, :40].cuda(),) * 2])
    before = cache.k.clone()
    for slots in (None, [0]):
        cache.evict(keep, 3, slots)
        assert torch.equal(cache.k, before) and cache.lengths.tolist() == [40] == [cache.length(0)] and cache.free_pages == 0


@pytest.mark.parametrize("top_k", LARGE + [-1, -2 ** 31, -2 ** 32 + 1])
def test_top_k(top_k):
    from complexity_deep_b200 import ops
    g = torch.Generator().manual_seed(3)
    x, u = torch.randn(8, 500, generator=g).cuda(), torch.rand(8, generator=g).cuda()
    for got, want in zip(ops.sample_tokens(x, u, 1.0, top_k, 0.9), ops.sample_tokens(x, u, 1.0, 0, 0.9)):
        assert torch.equal(got, want)
