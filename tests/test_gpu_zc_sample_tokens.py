"""Sampling from given numbers (cd_sample_tokens) against 64 bits.  The ids are whole numbers and must be equal: the kernel's masses
are exact sums of weights rounded to 2^-45, so a border between two tokens lies within V 2^-45 < 2^-27 of its place in units of the
largest weight, and the numbers here come no nearer to one by chance than some 2^-24.  A probability is rounded to fp32 (2^-24 of the
value, and 2^-27 for the sums)."""
import pytest
import torch

import paged_cases as cases

pytestmark = pytest.mark.gpu


def _check(x, u, t=1.0, k=0, p=1.0, m=0.0, rows=None):
    from complexity_deep_b200 import ops
    rules = [r.cuda() if isinstance(r, torch.Tensor) else r for r in (t, k, p, m)]
    ids, probs = ops.sample_tokens(x.cuda(), u.cuda(), *rules)
    ids2, probs2 = ops.sample_tokens(x.cuda(), u.cuda(), *rules)
    assert torch.equal(ids, ids2) and torch.equal(probs, probs2)
    f32 = lambda v, i: float(v[i] if isinstance(v, torch.Tensor) else torch.tensor(v, dtype=torch.float32))  # noqa: E731
    for i in range(x.shape[0]) if rows is None else rows:
        want, prob = cases.sample(x[i], float(u[i]), f32(t, i), int(k[i] if isinstance(k, torch.Tensor) else k), f32(p, i), f32(m, i))
        assert int(ids[i]) == want, (i, int(ids[i]), want)
        assert abs(float(probs[i]) - prob) <= 2.0 ** -23 * prob + 1e-12, (i, float(probs[i]), prob)


def _inputs(B, V, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    x = 2.0 * torch.randn(B, V, generator=g)
    x.scatter_(1, torch.randint(0, V, (B, min(V, 9)), generator=g), 6 + 2 * torch.randn(B, min(V, 9), generator=g))
    return x.to(dtype), torch.rand(B, generator=g)


RULES = [(1.0, 50, 0.9, 0.0), (0.7, 0, 1.0, 0.0), (1.3, 0, 0.5, 0.0), (1.0, 0, 1.0, 0.1), (0.9, 20, 0.95, 0.02), (0.0, 50, 0.9, 0.1),
         (1.0, 1, 1.0, 0.0), (1.0, 5000, 0.99, 0.0), (1e-3, 0, 0.9, 0.0), (50.0, 0, 0.9, 0.0), (1.0, 3, 1e-6, 0.0), (1.0, 0, 0.0, 1.0)]


@pytest.mark.parametrize("rules", RULES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_rules(rules, dtype):
    for V in (1000, 8191, 32000):
        _check(*_inputs(5, V, dtype, V + int(10 * rules[0])), *rules)


@pytest.mark.parametrize("V", [1, 2, 3, 31, 32, 33, 1023, 1024, 1025, 2048, 65537, 100000])
def test_vocabularies(V):
    for dtype in (torch.bfloat16, torch.float32):
        x, u = _inputs(3, V, dtype, V)
        for rules in ((1.0, 50, 0.9, 0.0), (1.0, 0, 0.9, 0.0), (0.0, 0, 1.0, 0.0)):
            _check(x, u, *rules)


@pytest.mark.parametrize("k", [192, 193, 200, 255, 256, 257, 511, 512, 513, 2047, 2048, 2049, 4999, 8191, 8192])
def test_sizes_of_top_k(k):
    """Around the largest k that takes the bound, the lists' sizes and the vocabulary."""
    for V in (8192, 50000):
        for dtype in (torch.bfloat16, torch.float32):
            x, u = _inputs(3, V, dtype, V + k)
            _check(x, u, 1.0, k, 0.9, 0.0)
            _check(x, u, 1.5, k, 1.0, 0.01)
    x = torch.randint(0, 50, (3, 9000), generator=torch.Generator().manual_seed(k)).to(torch.bfloat16)   # ties at every border
    _check(x, torch.rand(3, generator=torch.Generator().manual_seed(k)), 8.0, k, 0.8, 0.0)


def test_largest_vocabulary():
    x, u = _inputs(2, 1 << 18, torch.float32, 1)
    _check(x, u, 1.0, 0, 0.9, 0.0)
    _check(x, u, 1.0, 300, 0.9, 0.0)
    _check(torch.zeros(1, 1 << 18), torch.tensor([0.75]), 1.0, 0, 1.0, 0.0)    # the largest sum that there is


@pytest.mark.parametrize("B,V,dtype", [(75, 40960, torch.float32), (75, 40961, torch.float32), (75, 81920, torch.bfloat16),
                                       (38, 163840, torch.bfloat16), (37, 70000, torch.bfloat16), (20, 200000, torch.bfloat16)])
def test_shares_of_a_row(B, V, dtype):
    """The largest share that a block takes and one token more; rows whose clusters would not run at the same time."""
    x, u = _inputs(B, V, dtype, B)
    for rules in ((1.0, 0, 0.9, 0.0), (1.0, 3000, 0.99, 0.001), (0.8, 50, 0.9, 0.0)):
        _check(x, u, *rules, rows=(0, B // 2, B - 1))


def test_rules_by_row():
    x, u = _inputs(64, 5000, torch.float32, 5)
    g = torch.Generator().manual_seed(2)
    pick = lambda v: torch.tensor(v)[torch.randint(0, len(v), (64,), generator=g)]  # noqa: E731
    t, k, p, m = pick([0.0, 0.5, 1.0, 1.5]), pick([0, 1, 2, 50, 6000]).to(torch.int32), pick([0.3, 0.9, 1.0]), pick([0.0, 0.05, 0.5])
    _check(x, u, t, k, p, m)
    _check(x[:, 1:4001], u, t, 40, p, 0.0)                                     # rows apart, off a 16-byte boundary


def test_ties():
    """Few distinct values: which of the equal ones stay goes by their index, how many by the masses."""
    g = torch.Generator().manual_seed(3)
    x = torch.randint(0, 4, (6, 3000), generator=g).to(torch.bfloat16)
    u = torch.rand(6, generator=g)
    for rules in ((1.0, 10, 1.0, 0.0), (1.0, 10, 0.5, 0.0), (1.0, 0, 0.25, 0.0), (2.0, 1000, 0.75, 0.0), (1.0, 0, 0.9, 0.5)):
        _check(x, u, *rules)
    _check(torch.zeros(4, 64), torch.tensor([0.0, 0.2, 0.49, 0.999]), 1.0, 0, 0.5, 0.0)   # 33 of 64 have at most half ahead
    _check(torch.zeros(2, 64), torch.tensor([0.0, 0.5]), 0.0)


def test_borders():
    """u at the border between two equal tokens belongs to the second; 0 to the first that can be drawn, the largest u to the last."""
    x = torch.full((5, 40), -float("inf"))
    x[:, 7], x[:, 21] = 1.0, 1.0
    _check(x, torch.tensor([0.0, 0.49999997, 0.5, 0.50000006, 0.99999994]))


def test_infinities_and_nan():
    from complexity_deep_b200 import ops
    inf, nan = float("inf"), float("nan")
    x = torch.full((6, 300), -inf)
    x[0, 17] = 2.0                                     # one token left
    x[1, 5], x[1, 250] = inf, inf                      # two that outweigh everything
    x[1, 9] = 4.0
    x[2, :] = nan
    x[2, 100:110] = 1.0                                # NaN everywhere else
    x[3, :] = -inf                                     # nothing
    x[4, :] = nan
    x[5, :] = -3e38
    x[5, 50] = 3e38
    u = torch.tensor([0.9, 0.7, 0.55, 0.5, 0.5, 0.5])
    for rules in ((1.0, 0, 1.0, 0.0), (1.0, 50, 0.9, 0.0), (0.0, 0, 1.0, 0.0), (0.5, 3, 0.4, 0.3)):
        for dtype in (torch.float32, torch.bfloat16):
            _check(x.to(dtype), u, *rules)
    ids, probs = ops.sample_tokens(x[3:5].cuda(), u[:2].cuda())
    assert ids.tolist() == [0, 0] and probs.tolist() == [0.0, 0.0]


def test_small_values_and_zeros():
    """Zeros of both signs are equal; subnormal numbers and their neighbours are not."""
    g = torch.Generator().manual_seed(6)
    for dtype in (torch.bfloat16, torch.float32):
        pool = torch.tensor([0.0, -0.0, 1e-39, -1e-39, 2e-39, 1e-38, -3e-38, 1e-20]).to(dtype)
        x = pool[torch.randint(0, 8, (4, 1500), generator=g)]
        u = torch.rand(4, generator=g)
        for rules in ((1.0, 100, 1.0, 0.0), (1e-38, 0, 0.6, 0.0), (1e-20, 700, 0.5, 0.0), (2e-39, 0, 1.0, 0.2), (0.0, 0, 1.0, 0.0)):
            _check(x, u, *rules)


def test_odd_rules_and_strides():
    """Rules at the ends of their ranges and beyond, given numbers outside [0, 1), one row of logits for many draws."""
    from complexity_deep_b200 import ops
    nan, inf = float("nan"), float("inf")
    x, u = _inputs(1, 700, torch.float32, 4)
    many = torch.linspace(0, 0.999, 300)
    _check(x.expand(300, -1), many, 0.7, 30, 0.9, 0.0)
    assert ops.sample_tokens(x.cuda().expand(300, -1), many.cuda(), 0.7, 30, 0.9)[0].shape == (300,)
    best = int(x.argmax())
    for t in (0.0, -1.0, nan, 1e-30, 1e-37, 1e-40):                        # greedy, or so cold that only the largest has a weight
        ids, probs = ops.sample_tokens(x.cuda(), u.cuda(), t, 0, 0.9)
        assert ids.tolist() == [best] and probs.tolist() == [1.0], t
    want = ops.sample_tokens(x.cuda(), u.cuda())
    for rules in ((1.0, -3, 1.0, 0.0), (1.0, 700, 1.0, 0.0), (1.0, 10 ** 9, 2.0, -1.0), (1.0, 0, nan, nan), (1.0, 0, inf, 0.0)):
        assert torch.equal(ops.sample_tokens(x.cuda(), u.cuda(), *rules)[0], want[0]), rules
    assert int(ops.sample_tokens(x.cuda(), u.cuda(), inf)[0]) == int(float(u) * 700)     # all weigh the same
    ends = ops.sample_tokens(x.cuda().expand(5, -1), torch.tensor([-1.0, nan, 0.0, 1.0, 7.0]).cuda())[0].tolist()
    assert ends[0] == ends[1] == ends[2] == 0 and ends[3] == ends[4] == 699
    for p, m in ((0.0, 0.0), (-1.0, 0.0), (1.0, 1.0), (1.0, 5.0)):         # the largest alone
        assert ops.sample_tokens(x.cuda(), u.cuda(), 1.0, 0, p, m)[0].tolist() == [best]


def test_more_rows_than_a_grid_is_high():
    from complexity_deep_b200 import ops
    x = torch.zeros(70000, 8, device="cuda")
    x[:, 3] = 50.0
    x[69999, 3], x[69999, 5] = 0.0, 50.0
    ids, _ = ops.sample_tokens(x, torch.full((70000,), 0.5, device="cuda"))
    assert bool((ids[:-1] == 3).all()) and int(ids[-1]) == 5


def test_captured_and_empty():
    from complexity_deep_b200 import ops
    x, u = (t.cuda() for t in _inputs(3, 4000, torch.bfloat16, 8))
    graph = torch.cuda.CUDAGraph()
    ops.sample_tokens(x, u, 0.8, 40, 0.9)
    with torch.cuda.graph(graph):
        ids, probs = ops.sample_tokens(x, u, 0.8, 40, 0.9)
    for seed in range(3):
        a, b = _inputs(3, 4000, torch.bfloat16, 20 + seed)
        x.copy_(a), u.copy_(b)
        graph.replay()
        want = ops.sample_tokens(x, u, 0.8, 40, 0.9)
        assert torch.equal(ids, want[0]) and torch.equal(probs, want[1])
    assert ops.sample_tokens(x[:0], u[:0])[0].shape == (0,)
