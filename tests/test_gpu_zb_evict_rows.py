"""Eviction from a paged cache (cd_evict_rows): which rows stay and where they end up is decided by whole numbers and comparisons,
so everything must be equal to sorting in Python, bit for bit."""
import pytest
import torch

import paged_cases as cases

pytestmark = pytest.mark.gpu


def _run(lengths, hkv, D, page, keep, recent, seed=0, layers=None, order="heads", in_place=True, weights=None, ties=False, width=None):
    from complexity_deep_b200 import ops
    k, v, table = cases.make_cache(lengths, hkv, D, page, seed, layers=layers, order=order, width=width)
    g = torch.Generator().manual_seed(seed + 1)
    B, rows = len(lengths), table.shape[1] * page
    shape = ((layers,) if layers else ()) + (B, hkv, rows)
    if weights is None:
        weights = torch.randint(0, 5, shape, generator=g).float() if ties else torch.randn(shape, generator=g).exp()
    pos = torch.rand(shape, generator=g).argsort(-1).to(torch.int32)          # any order: earlier evictions have mixed the rows
    nxt = torch.tensor([max(0, n) for n in lengths], dtype=torch.int32) + 3
    dev = lambda t: t.cuda() if t.is_contiguous() else t.transpose(-3, -2).cuda().transpose(-3, -2)  # noqa: E731
    kd, vd, wd, pd = dev(k), dev(v), weights.cuda(), pos.cuda()
    w_out, p_out = (wd, pd) if in_place else (torch.full_like(wd, 7.0), torch.full_like(pd, 7))
    extra = {} if in_place else {"weights_out": w_out, "row_positions_out": p_out}
    n = torch.tensor(lengths, dtype=torch.int32).cuda()
    ops.evict_rows_(kd, vd, table.cuda(), n, nxt.cuda(), wd, pd, keep, recent, **extra)
    ops.status_fetch()
    want_w, want_p = (weights.clone(), pos.clone()) if in_place else (torch.full_like(weights, 7.0), torch.full_like(pos, 7))
    want = [k.clone(memory_format=torch.preserve_format), v.clone(memory_format=torch.preserve_format)]
    for layer in range(layers or 1):
        pick = (lambda t: t[layer]) if layers else (lambda t: t)
        for b, m in enumerate(lengths):
            for h in range(hkv):
                src = cases.evict(pick(weights)[b, h].tolist(), pick(pos)[b, h].tolist(), max(0, m), int(nxt[b]) - recent, keep)
                for to, s in enumerate(src):
                    pick(want_w)[b, h, to], pick(want_p)[b, h, to] = pick(weights)[b, h, s], pick(pos)[b, h, s]
                    if to != s:
                        for pool, old in zip(want, (k, v)):
                            pick(pool)[table[b, to // page], h, to % page] = pick(old)[table[b, s // page], h, s % page]
    assert torch.equal(w_out.cpu().view(torch.int32), want_w.view(torch.int32)) and torch.equal(p_out.cpu(), want_p)
    for got, ref in zip((kd, vd), want):
        got, ref = (t.cpu().transpose(-3, -2).contiguous() if order == "rows" else t.cpu() for t in (got, ref))
        assert torch.equal(got.view(torch.int16), ref.view(torch.int16))
    if not in_place:
        assert torch.equal(wd.cpu().view(torch.int32), weights.view(torch.int32)) and torch.equal(pd.cpu(), pos)


@pytest.mark.parametrize("in_place", [True, False])
@pytest.mark.parametrize("page,D", [(16, 64), (64, 128), (256, 64), (5, 8), (1, 128)])
def test_pages_and_heads(page, D, in_place):
    _run([300, 256, 257, 0, 1, 299], 2, D, page, 256, 32, seed=page, in_place=in_place)
    _run([130, 77], 3, D, page, 40, 0, seed=page, in_place=in_place, order="rows", ties=True)


@pytest.mark.parametrize("keep,recent", [(1, 0), (1, 1), (2, 1), (63, 63), (64, 10), (99, 50), (100, 0), (101, 5), (5000, 7)])
def test_budgets(keep, recent):
    _run([100, 99, -1], 2, 64, 16, keep, recent, seed=keep)
    _run([100, 64], 1, 64, 16, keep, recent, seed=keep, ties=True, in_place=False)


def test_layers_and_long():
    _run([200, 150], 2, 64, 16, 64, 8, seed=3, layers=3)
    _run([200, 150], 2, 64, 16, 64, 8, seed=3, layers=2, order="rows", in_place=False)
    _run([33000, 5], 1, 64, 128, 4000, 100, seed=4)
    _run([33000], 1, 64, 128, 30000, 100, seed=5, ties=True)
    _run([40 + i for i in range(50)], 8, 64, 16, 41, 4, seed=6)


def test_rows_beyond_what_a_block_holds():
    """Shares of more than 49 152 rows: keys are read again, lists lie in the workspace; also with several blocks a pair."""
    _run([60000, 700], 1, 64, 256, 650, 100, seed=7, width=256)
    _run([3000, 60000, 64], 2, 8, 64, 2000, 0, seed=8, width=1024, in_place=False)
    _run([60000], 1, 64, 64, 30000, 5, seed=9, width=1000, ties=True, order="rows")
    _run([700, 60000, 50, 3], 40, 8, 64, 600, 3, seed=10, width=1024, ties=True)          # one block a pair


@pytest.mark.parametrize("rows,keep", [(520, 256), (2100, 1050), (4200, 300), (9000, 4500), (17000, 16000), (33000, 1)])
@pytest.mark.parametrize("ties", [False, True])
def test_several_blocks_a_pair(rows, keep, ties):
    """Clusters of 2 to 8 blocks: shares of rows that end anywhere, equal weights across their borders, sequences shorter than the
    table (blocks without rows), both ways of writing the outputs."""
    _run([rows, rows // 2, 3, keep + 1], 1, 8, 16, keep, 1, seed=rows, ties=ties, in_place=ties)
    _run([rows - 7], 3, 16, 32, keep, keep // 3, seed=keep, ties=ties, in_place=not ties, width=-(-rows // 32) + 9)


@pytest.mark.parametrize("pairs,rows", [(16, 9000), (36, 5000), (149, 400), (149, 3990), (149, 4100), (600, 200), (600, 2600), (600, 60)])
def test_many_pairs(pairs, rows):
    """Pairs whose clusters would not all run together, more pairs than SMs, and than four an SM: blocks of 128, 256 and 1 024 threads."""
    from complexity_deep_b200 import ops
    g = torch.Generator().manual_seed(rows)
    width = -(-rows // 16)
    pool = torch.randn(pairs * width, 1, 16, 8, generator=g).to(torch.bfloat16).cuda()
    table = torch.arange(pairs * width, dtype=torch.int32, device="cuda").view(pairs, width)
    w, pos = torch.randn(pairs, 1, width * 16, generator=g).exp(), torch.rand(pairs, 1, width * 16, generator=g).argsort(-1).to(torch.int32)
    keep, n = rows // 2, torch.full((pairs,), rows, dtype=torch.int32, device="cuda")
    wd, pd, kd, vd = w.cuda(), pos.cuda(), pool.clone(), pool.clone() + 1
    ops.evict_rows_(kd, vd, table, n, n, wd, pd, keep, 7)
    flat, moved = pool.view(pairs, width * 16, 8).cpu(), kd.view(pairs, width * 16, 8).cpu()
    for b in list(range(0, pairs, 37)) + [pairs - 1]:
        src = torch.tensor(cases.evict(w[b, 0].tolist(), pos[b, 0].tolist(), rows, rows - 7, keep))
        assert torch.equal(moved[b, :keep], flat[b, src]) and torch.equal(moved[b, keep:], flat[b, keep:])
        assert torch.equal(wd[b, 0, :keep].cpu(), w[b, 0, src]) and torch.equal(pd[b, 0, :keep].cpu(), pos[b, 0, src])
    assert torch.equal(vd.view(pairs, width * 16, 8).cpu()[:, :keep], (moved + 1)[:, :keep])


def test_odd_weights():
    """Equal ones, zeros of both signs, negative, infinite and NaN."""
    shape = (2, 1, 160)
    _run([150, 160], 1, 64, 16, 70, 9, weights=torch.ones(shape))
    g = torch.Generator().manual_seed(1)
    pool = torch.tensor([0.0, -0.0, 1.0, -3.0, float("inf"), -float("inf"), float("nan"), 1e-40, 3e38])
    w = pool[torch.randint(0, 9, shape, generator=g)]
    for keep in (20, 70, 120, 149):
        _run([150, 160], 1, 64, 16, keep, 9, weights=w)


def test_rows_behind_the_end_do_not_count():
    """Large weights left behind by an earlier sequence, NaN in the rows themselves (make_cache puts them there)."""
    w = torch.rand(1, 2, 256)
    w[:, :, 100:] = 1e9
    _run([100], 2, 64, 16, 60, 5, weights=w, width=16)


def test_captured():
    """A captured call follows weights and lengths that change between replays."""
    from complexity_deep_b200 import ops
    k, v, table = (t.cuda() for t in cases.make_cache([160, 160], 2, 64, 16, 2))
    w, pos = torch.rand(2, 2, 160, device="cuda"), torch.arange(160, dtype=torch.int32, device="cuda").expand(2, 2, 160).contiguous()
    n, nxt = torch.tensor([160, 160], dtype=torch.int32).cuda(), torch.tensor([160, 160], dtype=torch.int32).cuda()
    wo, po = torch.zeros_like(w), torch.zeros_like(pos)
    call = lambda kk, vv, a, b: ops.evict_rows_(kk, vv, table, n, nxt, w, pos, 50, 5, weights_out=a, row_positions_out=b)  # noqa: E731
    call(k.clone(), v.clone(), wo, po)
    kg, vg = k.clone(), v.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(kg, vg, wo, po)
    for lens in ([160, 160], [49, 120], [51, 0]):
        n.copy_(torch.tensor(lens, dtype=torch.int32))
        w.uniform_()
        kg.copy_(k), vg.copy_(v)
        graph.replay()
        ke, ve, we, pe = k.clone(), v.clone(), torch.zeros_like(w), torch.zeros_like(pos)
        call(ke, ve, we, pe)
        held = torch.arange(160, device="cuda") < n.clamp(max=50)[:, None, None]
        assert torch.equal(torch.where(held, wo, 0), we) and torch.equal(torch.where(held, po, 0), pe)
        assert torch.equal(kg.view(torch.int16), ke.view(torch.int16)) and torch.equal(vg.view(torch.int16), ve.view(torch.int16))


def test_bad_page_is_skipped():
    from complexity_deep_b200 import ops, _lib
    k, v, table = cases.make_cache([64], 1, 64, 16, 1, rest=0.0)
    table[0, 3] = -1
    w = torch.arange(64, dtype=torch.float32).view(1, 1, 64).cuda()          # the last rows weigh most: they would move
    pos, n = torch.zeros(1, 1, 64, dtype=torch.int32).cuda(), torch.tensor([64], dtype=torch.int32).cuda()
    ops.evict_rows_(k.cuda(), v.cuda(), table.cuda(), n, n, w, pos, 16, 0)
    with pytest.raises(_lib.CdeepError):
        ops.status_fetch()
    ops.status_fetch()


def test_length_beyond_the_table_is_refused():
    from complexity_deep_b200 import ops, _lib
    k, v, table = cases.make_cache([64, 64], 1, 64, 16, 1, rest=0.0)
    w, pos = torch.rand(2, 1, 64).cuda(), torch.zeros(2, 1, 64, dtype=torch.int32).cuda()
    before, n, kd = w.clone(), torch.tensor([65, 40], dtype=torch.int32).cuda(), k.cuda()
    ops.evict_rows_(kd, v.cuda(), table.cuda(), n, n, w, pos, 16, 0)
    with pytest.raises(_lib.CdeepError):
        ops.status_fetch()
    assert torch.equal(w[0], before[0]) and not torch.equal(w[1], before[1])
    mine = table[0].long()
    assert torch.equal(kd[mine.cuda()].cpu(), k[mine])
    assert ops.evict_rows_(kd, kd, table[:0].cuda(), n[:0], n[:0], w[:0], pos[:0], 16, 0) is None
