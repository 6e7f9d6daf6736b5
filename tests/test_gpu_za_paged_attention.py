"""Attention over a paged cache (cd_paged_attention, cd_paged_step_attention) against 64 bits.

What a result may be off by: the output is rounded to bf16 (half a step, 2^-8 of the value); a score is a sum of D products in 32
bits, |error| <= D 2^-24 sum|q k| / sqrt(D) <= 2^-14 for the normal inputs here, which moves a weight by twice that, so an output
by 2^-12 sum p|v| and a weight by 2^-12 of itself (the weights of a head's rows are held as two bf16 numbers, 2^-16).  In a step
q keeps 16 bits: 2^-17 sum|q k| / sqrt(D) <= 2^-13 on a score, hence 2^-11.  Rows behind a sequence's end and pages that
nobody has are NaN in every test."""
import pytest
import torch

import paged_cases as cases

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def _close(out, ref, size, loose):
    bad = (out.double().cpu() - ref).abs() > 2.0 ** -8 * ref.abs() + loose * size
    assert not bool(bad.any()) and bool(torch.isfinite(out).all())


def _attend(lengths, hkv, G, D, page, seed=0, weights=False, **kw):
    from complexity_deep_b200 import ops
    k, v, table = cases.make_cache(lengths, hkv, D, page, seed, **kw)
    g = torch.Generator().manual_seed(seed + 1)
    B, hq, rows = len(lengths), hkv * G, table.shape[1] * page
    q = torch.randn(B, (hq + 2 * hkv) * D, generator=g).to(BF)
    old = torch.rand(B, hkv, rows, generator=g) if weights else None
    acc = old.cuda() if weights else None
    n = torch.tensor(lengths, dtype=torch.int32)
    dev = lambda t: t.cuda() if t.is_contiguous() else t.transpose(1, 2).cuda().transpose(1, 2)  # noqa: E731
    out = ops.paged_attention(q.cuda(), dev(k), dev(v), table.cuda(), n.cuda(), hq, hkv, D, weights=acc)
    ops.status_fetch()
    ref, size, share = cases.attend(q[:, : hq * D].double().view(B, hq, D), k, v, table, lengths, hkv)
    _close(out.view(B, hq, D), ref, size, 2.0 ** -12)
    if weights:
        for b, m in enumerate(lengths):
            m = max(0, m)
            got, want = acc[b].double().cpu(), old[b].double()
            off = (got[:, :m] - want[:, :m] - share[b]).abs()
            assert bool((off <= 2.0 ** -12 * share[b] + 2.0 ** -23 * (want[:, :m] + share[b])).all())
            assert torch.equal(got[:, m:], want[:, m:])                   # rows behind the end stay as they were


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("G,D", [(1, 64), (2, 128), (3, 64), (4, 128), (7, 128), (8, 64), (9, 64), (16, 128)])
def test_groups_and_pages(G, D, page):
    _attend([1, page - 1, page, page + 1, 0, 331, 64, 65], 2, G, D, page, seed=page + G, weights=G % 2 == 0)


@pytest.mark.parametrize("lengths", [[1], [2], [15], [16], [17], [63], [64], [65], [128], [4097], [0], [0, 0, 5], [20000, 1, 700]])
@pytest.mark.parametrize("weights", [False, True])
def test_lengths(lengths, weights):
    _attend(lengths, 4, 2, 128, 64, seed=len(lengths) + lengths[0], weights=weights)
    _attend(lengths, 1, 3, 64, 16, seed=lengths[0], weights=weights, order="rows")


def test_long_and_many():
    _attend([33000, 12], 1, 2, 128, 128, seed=5, weights=True)
    _attend([70] * 150, 8, 2, 64, 16, seed=6, weights=True)
    _attend([(37 * i) % 500 for i in range(70)], 3, 4, 128, 32, seed=7, weights=True, order="rows")
    _attend([-1, 9, -1], 2, 2, 64, 16, seed=8, weights=True)


@pytest.mark.parametrize("G,D", [(1, 128), (3, 64), (8, 128), (9, 64), (16, 128), (16, 64)])
@pytest.mark.parametrize("weights", [False, True])
def test_line_of_tiles(G, D, weights):
    """More tiles than clusters take: pairs cut between many blocks, several pairs a block, sequences without rows in between."""
    _attend([20000, 1, 0, 700], 2, G, D, 64, seed=G, weights=weights)
    _attend([0] + [(97 * i) % 260 for i in range(130)] + [0], 3, G, D, 16, seed=G + 1, weights=weights, order="rows")


@pytest.mark.parametrize("G,D", [(1, 64), (2, 128), (5, 64), (16, 128)])
@pytest.mark.parametrize("lengths", [[19000], [15000, 9000, 40], [2600] * 17])
def test_pairs_cut_between_most_blocks(lengths, G, D):
    """One head of keys: a part of a pair from hundreds of blocks, from about a hundred, from some twenty."""
    _attend(lengths, 1, G, D, 64, seed=G, weights=G % 2 == 1)


@pytest.mark.parametrize("G,D", [(2, 128), (16, 128), (3, 64)])
@pytest.mark.parametrize("weights", [False, True])
def test_many_short_pairs_beside_long_ones(G, D, weights):
    """Pairs of a tile each, whose beginnings are most of what a block has, ahead of, behind and between long ones; stretches that lie
    within a pair's beginning."""
    _attend([3000] * 6 + [1, 64, 0, 65] * 15 + [2500], 2, G, D, 64, seed=G, weights=weights)
    _attend([5] * 40 + [9000] + [0, 70] * 20, 5, G, D, 16, seed=G + 1, weights=weights, order="rows")
    _attend([1100], 1, G, D, 64, seed=G + 2, weights=weights)
    _attend([(53 * i) % 211 * (i % 5 > 0) for i in range(450)], 2, G, D, 16, seed=G + 4, weights=weights)     # several sequences a thread
    _attend([9, 0, 9000, 9], 1, G, D, 64, seed=G + 3, weights=weights)


def test_strides_and_shared_pages():
    """Pools that are every other page and a part of the heads of larger ones, a table that is a part of a wider one, two
    sequences that share their first pages."""
    from complexity_deep_b200 import ops
    k, v, table = cases.make_cache([300, 300, 77], 2, 128, 32, 3)
    table[1, :5] = table[0, :5]
    big = [torch.full((2 * k.shape[0], 5, 32, 128), float("nan"), dtype=BF, device="cuda") for _ in range(2)]
    for pool, t in zip(big, (k, v)):
        pool[::2, 1:3] = t.cuda()
    wide = torch.full((3, 40), -7, dtype=torch.int32, device="cuda")
    wide[:, : table.shape[1]] = table.cuda()
    q = torch.randn(3, 4 * 128, generator=torch.Generator().manual_seed(1)).to(BF)
    n = torch.tensor([300, 290, 77], dtype=torch.int32, device="cuda")
    out = ops.paged_attention(q.cuda(), big[0][::2, 1:3], big[1][::2, 1:3], wide[:, : table.shape[1]], n, 4, 2, 128)
    ref, size, _ = cases.attend(q.double().view(3, 4, 128), k, v, table, [300, 290, 77], 2)
    _close(out.view(3, 4, 128), ref, size, 2.0 ** -12)


def test_large_scores_and_equal_ones():
    """Scores in the hundreds (one row takes everything), all alike, and growing along the cache."""
    from complexity_deep_b200 import ops
    D, n = 64, 1000
    k, v, table = cases.make_cache([n], 1, D, 16, 9)
    q = torch.randn(1, D, generator=torch.Generator().manual_seed(2)).to(BF)
    for scale in (0.0, 30.0):
        kk = (k.float() * scale).to(BF)
        out = ops.paged_attention(q.cuda(), kk.cuda(), v.cuda(), table.cuda(), torch.tensor([n], dtype=torch.int32).cuda(), 1, 1, D)
        ref, size, _ = cases.attend(q.double().view(1, 1, D), kk, v, table, [n], 1)
        _close(out.view(1, 1, D), ref, size, 2.0 ** -9)                    # scores 30 times as large, errors too
    rising = torch.zeros_like(k)
    for r in range(n):
        rising[table[0, r // 16], 0, r % 16] = (q[0].float() / q.float().norm() * r * 0.05).to(BF)
    out = ops.paged_attention(q.cuda(), rising.cuda(), v.cuda(), table.cuda(), torch.tensor([n], dtype=torch.int32).cuda(), 1, 1, D)
    ref, size, _ = cases.attend(q.double().view(1, 1, D), rising, v, table, [n], 1)
    _close(out.view(1, 1, D), ref, size, 2.0 ** -9)


def test_not_finite():
    """A NaN key or value that is seen makes its heads NaN and no others'."""
    from complexity_deep_b200 import ops
    k, v, table = cases.make_cache([100, 100], 2, 64, 16, 4)
    q = torch.randn(2, 4 * 64, generator=torch.Generator().manual_seed(3)).to(BF).cuda()
    n = torch.tensor([100, 100], dtype=torch.int32).cuda()
    clean = ops.paged_attention(q, k.cuda(), v.cuda(), table.cuda(), n, 4, 2, 64).view(2, 2, 2, 64)
    for pool in (k, v):
        bad = pool.clone()
        bad[table[1, 6], 1, 3, 5] = float("nan")                           # row 99 of sequence 1
        args = (bad.cuda(), v.cuda()) if pool is k else (k.cuda(), bad.cuda())
        out = ops.paged_attention(q, *args, table.cuda(), n, 4, 2, 64).view(2, 2, 2, 64)
        assert bool(out[1, 1].isnan().all() if pool is k else out[1, 1, :, 5].isnan().all())
        assert torch.equal(out[0], clean[0]) and torch.equal(out[1, 0], clean[1, 0])


def _step(lengths, hkv, G, D, page, seed=0, norm=True, weights=False, order="heads", ahead=7):
    from complexity_deep_b200 import ops
    k, v, table = cases.make_cache(lengths, hkv, D, page, seed, room=1, order=order)
    g = torch.Generator().manual_seed(seed + 1)
    B, hq, rows = len(lengths), hkv * G, table.shape[1] * page
    qkv = torch.randn(B, (hq + 2 * hkv) * D, generator=g).to(BF)
    qw, kw = ((1 + 0.2 * torch.randn(2, D, generator=g)).to(BF)) if norm else (None, None)
    cos, sin = cases.tables(rows + ahead + 1, D)
    n, pos = torch.tensor(lengths, dtype=torch.int32), torch.tensor([m + ahead for m in lengths], dtype=torch.int32)
    old = torch.rand(B, hkv, rows, generator=g)
    acc, where = (old.cuda(), torch.full((B, hkv, rows), -5, dtype=torch.int32).cuda()) if weights else (None, None)
    dev = lambda t: None if t is None else t.cuda() if t.is_contiguous() else t.transpose(1, 2).cuda().transpose(1, 2)  # noqa: E731
    kd, vd, qd = dev(k), dev(v), qkv.cuda()
    args = (qd, dev(qw), dev(kw), cos.cuda(), sin.cuda(), cases.EPS, hq, hkv, D, kd, vd, table.cuda(), n.cuda(), pos.cuda())
    out = ops.paged_step_attention(*args, weights=acc, row_positions=where)
    ops.status_fetch()
    assert torch.equal(qd.cpu(), qkv)
    heads = qkv.double().view(B, hq + 2 * hkv, D)
    q = torch.zeros(B, hq, D, dtype=torch.float64)
    k1, v1 = kd.cpu(), vd.cpu()
    for b, m in enumerate(lengths):
        if m < 0:
            continue
        q[b] = cases.rotate(heads[b, :hq], qw, cos[m + ahead], sin[m + ahead])
        key = cases.rotate(heads[b, hq:hq + hkv], kw, cos[m + ahead], sin[m + ahead])
        to = (table[b, m // page], slice(None), m % page)
        got = k1[to].double()
        # a rounding to bf16 behind some ten operations in 32 bits
        assert bool(((got - key).abs() <= 2.0 ** -8 * key.abs() + 2.0 ** -19 * key.abs().max()).all())
        assert torch.equal(v1[to], qkv.view(B, -1, D)[b, hq + hkv:])
        k[to], v[to] = k1[to], v1[to]
    same = lambda a, b: torch.equal(a.view(torch.int16), b.view(torch.int16)) if a.is_contiguous() else same(a.transpose(1, 2), b.transpose(1, 2))  # noqa: E731
    assert same(k1, k) and same(v1, v)                                     # nothing else has been written
    after = [m + 1 if m >= 0 else 0 for m in lengths]
    ref, size, share = cases.attend(q, k, v, table, after, hkv)
    _close(out.view(B, hq, D), ref, size, 2.0 ** -11)
    if weights:
        for b, m in enumerate(lengths):
            want = old[b].double()
            if m >= 0:
                want[:, m] = 0.0
            want[:, : after[b]] += share[b]
            off = (acc[b].double().cpu() - want).abs()
            loose = torch.zeros_like(want)
            loose[:, : after[b]] = share[b]
            assert bool((off <= 2.0 ** -11 * loose + 2.0 ** -23 * want).all())
            there = where[b].cpu()
            assert (there != -5).sum() == (hkv if m >= 0 else 0)
            if m >= 0:
                assert bool((there[:, m] == m + ahead).all())


@pytest.mark.parametrize("G,D,page", [(1, 128, 16), (2, 128, 64), (3, 64, 16), (4, 64, 256), (8, 128, 32), (16, 64, 64), (11, 128, 128)])
@pytest.mark.parametrize("order", ["heads", "rows"])
def test_step(G, D, page, order):
    _step([0, 1, page - 1, page, 200, -1, 63, 64, 127], 2, G, D, page, seed=G, weights=G != 2, order=order)


@pytest.mark.parametrize("norm", [False, True])
def test_step_sizes(norm):
    _step([0], 1, 1, 64, 16, norm=norm, weights=True)
    _step([-1], 1, 2, 64, 16, norm=norm, weights=True)
    _step([300], 4, 3, 64, 16, norm=norm)
    _step([6000, 3], 8, 2, 128, 64, norm=norm, weights=True)
    _step([(53 * i) % 400 - 1 for i in range(40)], 8, 2, 128, 64, norm=norm, weights=True)


@pytest.mark.parametrize("G,D", [(2, 64), (4, 128), (12, 64), (16, 128)])
def test_step_on_a_line_of_tiles(G, D):
    _step([20000, -1, 3, 639, 640], 2, G, D, 64, seed=G, weights=True)
    _step([(97 * i) % 260 - 1 for i in range(130)], 3, G, D, 16, seed=G + 1, weights=True, order="rows")


def test_no_room_and_bad_tables():
    """A full sequence, a position without a rotation and a page outside the pool are refused on the device: zeros, nothing
    stored, the status word raised; the other sequences are as ever."""
    from complexity_deep_b200 import ops, _lib
    k, v, table = cases.make_cache([31, 20, 20, 20], 2, 64, 16, 11, room=1, rest=0.0, width=2)
    g = torch.Generator().manual_seed(1)
    qkv = torch.randn(4, 8 * 64, generator=g).to(BF).cuda()
    cos, sin = (t.cuda() for t in cases.tables(40, 64))
    call = lambda n, pos, t, kd, vd: ops.paged_step_attention(  # noqa: E731
        qkv, None, None, cos, sin, 1e-6, 4, 2, 64, kd, vd, t, torch.tensor(n, dtype=torch.int32).cuda(),
        torch.tensor(pos, dtype=torch.int32).cuda())
    kd, vd, td = k.cuda(), v.cuda(), table.cuda()
    good = call([31, 20, 20, 20], [31, 20, 20, 20], td, kd, vd)
    ops.status_fetch()
    kd, vd, bad = k.cuda(), v.cuda(), table.clone()
    bad[2, 1] = k.shape[0]
    out = call([32, 20, 20, 20], [32, 40, 20, 20], bad.cuda(), kd, vd)
    with pytest.raises(_lib.CdeepError):
        ops.status_fetch()
    assert bool((out[:3] == 0).all()) and torch.equal(out[3], good[3])
    keep = torch.ones(k.shape[0], dtype=torch.bool)
    keep[table[3, 1]] = False
    assert torch.equal(kd.cpu()[keep], k[keep]) and torch.equal(vd.cpu()[keep], v[keep])
    out = ops.paged_attention(qkv, kd, vd, bad.cuda(), torch.tensor([16, 33, 20, 16], dtype=torch.int32).cuda(), 4, 2, 64)
    with pytest.raises(_lib.CdeepError):
        ops.status_fetch()
    assert bool((out[1] == 0).all())
    ops.status_fetch()


def test_refusals():
    from complexity_deep_b200 import ops
    k, v, table = (t.cuda() for t in cases.make_cache([40, 40], 2, 64, 16, 1, room=1, rest=0.0))
    q, n = torch.zeros(2, 8 * 64, dtype=BF, device="cuda"), torch.tensor([40, 40], dtype=torch.int32, device="cuda")
    cos, sin = (t.cuda() for t in cases.tables(64, 64))
    rows = table.shape[1] * 16
    w = torch.zeros(2, 2, rows, device="cuda")
    good = dict(q=q, k_pages=k, v_pages=v, block_table=table, lengths=n, hq=4, hkv=2, head_dim=64)
    ops.paged_attention(**good)
    odd = torch.zeros(2 * 2 * rows + 1, device="cuda")[1:].view(2, 2, rows)              # not on an 8-byte boundary
    for bad in (dict(q=q.float()), dict(q=q[:, :255]), dict(q=q[:, 1:]), dict(k_pages=k.float()), dict(k_pages=k[:, :1]), dict(v_pages=v[:3]),
                dict(k_pages=k.transpose(2, 3)), dict(block_table=table.long()), dict(block_table=table[:1]), dict(lengths=n.long()),
                dict(lengths=n[:1]), dict(lengths=n.cpu()), dict(block_table=table.cpu()), dict(hq=3), dict(hq=34), dict(head_dim=32),
                dict(weights=w[:, :1]), dict(weights=w.double()), dict(weights=odd), dict(k_pages=k[:, :, :12], v_pages=v[:, :, :12])):
        with pytest.raises(Exception) as e:
            ops.paged_attention(**{**good, **bad})
        assert isinstance(e.value, RuntimeError), bad
    step = dict(qkv=q, q_w=None, k_w=None, cos=cos, sin=sin, eps=1e-6, hq=4, hkv=2, head_dim=64, k_pages=k, v_pages=v, block_table=table,
                lengths=n, positions=n)
    ops.paged_step_attention(**step)
    one = torch.ones(64, dtype=BF, device="cuda")
    for bad in (dict(qkv=q[:, :256]), dict(q_w=one), dict(k_w=one), dict(q_w=one[:32], k_w=one), dict(cos=cos[:, :32]), dict(sin=sin[:9]),
                dict(cos=cos.double()), dict(positions=n.long()), dict(row_positions=w)):
        with pytest.raises(RuntimeError):
            ops.paged_step_attention(**{**step, **bad})
    assert ops.paged_attention(q[:0], k, v, table[:0], n[:0], 4, 2, 64).shape == (0, 256)
    # tables and weights off their boundaries are taken all the same
    shifted = torch.empty(64 * 64 + 1, device="cuda")[1:].view(64, 64).copy_(cos)
    w1 = torch.ones(65, dtype=BF, device="cuda")[1:]
    a = ops.paged_step_attention(**{**step, "q_w": one, "k_w": one})
    assert torch.equal(a, ops.paged_step_attention(**{**step, "cos": shifted, "q_w": w1, "k_w": w1}))


def test_captured_and_streams():
    """A captured step follows lengths that change between replays; two graphs and an eager call share nothing."""
    from complexity_deep_b200 import ops
    k, v, table = cases.make_cache([900, 40], 4, 128, 64, 12)
    q = torch.randn(2, 8 * 128, generator=torch.Generator().manual_seed(4)).to(BF).cuda()
    kd, vd, td = k.cuda(), v.cuda(), table.cuda()
    n = torch.tensor([900, 40], dtype=torch.int32).cuda()
    acc = [torch.zeros(2, 4, table.shape[1] * 64, device="cuda") for _ in range(2)]
    ops.paged_attention(q, kd, vd, td, n, 8, 4, 128, weights=acc[0])
    graphs, outs = [], []
    for a in acc:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(ops.paged_attention(q, kd, vd, td, n, 8, 4, 128, weights=a))
    side = [torch.cuda.Stream() for _ in range(2)]
    for lens in ([900, 40], [1, 0], [513, 39]):
        n.copy_(torch.tensor(lens, dtype=torch.int32))
        for a in acc:
            a.zero_()
        torch.cuda.synchronize()
        for s, graph in zip(side, graphs):
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        want = torch.zeros_like(acc[0])
        eager = ops.paged_attention(q, kd, vd, td, n, 8, 4, 128, weights=want)
        for o, a in zip(outs, acc):
            assert torch.equal(o, eager) and torch.equal(a, want)
