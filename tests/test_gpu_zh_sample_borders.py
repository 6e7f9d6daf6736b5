"""Borders that lie within 2^-30.4 to 2^-30 of the mass: n tokens of weight w = exp(x) against m of weight 1, where n w is that little more
than m.  Weights are good to 2^-30.6 of themselves (their sums are exact), so the heavier side is known; weights that are cut off
behind 2^-30 put it on the other one."""
import pytest
import torch

import paged_cases as cases

pytestmark = pytest.mark.gpu

BORDERS = [(305, 297, "-0x1.b37b14p-6"), (585, 407, "-0x1.73817ep-2"), (250, 147, "-0x1.0fe2f2p-1"), (329, 303, "-0x1.5133f6p-4"),
           (275, 94, "-0x1.12cf58p+0"), (490, 477, "-0x1.b88c38p-6"), (398, 321, "-0x1.b857a0p-3"), (317, 145, "-0x1.907854p-1"),
           (407, 234, "-0x1.1b6350p-1"), (367, 357, "-0x1.c4a01ep-6"), (312, 217, "-0x1.73d204p-2"), (562, 299, "-0x1.431a12p-1"),
           (235, 129, "-0x1.331576p-1"), (485, 244, "-0x1.5fbbeep-1")]


@pytest.mark.parametrize("V", [1000, 9000, 70000])
@pytest.mark.parametrize("k", [0, 2000])
def test_borders_of_equal_sides(V, k):
    from complexity_deep_b200 import ops
    rows, us, ps = [], [], []
    inf = float("inf")
    for n, m, x in BORDERS:
        light, heavy = torch.full((n,), float.fromhex(x)), torch.zeros(m)
        behind = torch.full((V - n - m,), -inf)
        rows += [torch.cat([light, behind, heavy]), torch.cat([heavy, behind, light]), torch.cat([heavy, light, behind])]
        us += [0.5, 0.5, 0.99999994]
        ps += [1.0, 1.0, 0.5]                                # the last: a light one is in the nucleus, as m is no more than half
    x, u, p = torch.stack(rows), torch.tensor(us), torch.tensor(ps)
    ids, probs = ops.sample_tokens(x.cuda(), u.cuda(), 1.0, k, p.cuda(), 0.0)
    want = []
    for i, (n, m, _) in enumerate(BORDERS):
        want += [n - 1, V - n, m]
    assert ids.tolist() == want
    for i in range(0, len(want), 5):
        assert cases.sample(x[i], us[i], 1.0, k, ps[i], 0.0)[0] == want[i]
