"""Sums over a long cache: additions that cut off what 32 bits do not hold, instead of rounding it, add up over hundreds of tiles."""
import pytest
import torch

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


@pytest.mark.parametrize("G,D", [(1, 64), (8, 64), (2, 128), (8, 128), (16, 64), (16, 128)])
def test_values_that_cancel(G, D):
    """Values between 1/2 and 1 in the first half of 16 384 rows, the same with the other sign (and the same keys, in the same order) in the
    second: what is left of a column is the errors of its sums, which rise to S and fall again.  A warp adds some 256 products of 16 rows
    to S <= 2 048 (4 warps: a quarter of 8 192 rows of weight and value up to 1 each, and what the largest weights leave of the
    others).  Rounded to 24 bits, each addition is off by up to 2^-14 S / 2 048 either way, 0.29 steps of 2^-13 on average: 4 x 256 of them 32 x
    0.29 x 2^-13 = 2^-9.8, in units of the sum of weights, 16 384 e^-1 at least for the scores here, 2^-22.4.  Ten times that is
    2^-19; a cut of half a step towards zero each time is 4 x 256 x 2^-14 / 2^12.6 = 2^-16.6, always to the same side.  More than eight heads
    add inside of the products, three a tile: 4 x 256 x 3 x 2^-12 / 2^12.6 = 2^-13 at worst.  64 sequences share the pages, so that a block's
    stretch has hundreds of tiles; the last ones are cut between blocks."""
    from complexity_deep_b200 import ops
    B, hkv, page, rows = 64, 8 if D == 64 else 6, 64, 16384
    g = torch.Generator().manual_seed(G + D)
    half = rows // 2 // page
    k = (0.25 * torch.randn(half, hkv, page, D, generator=g)).to(BF)
    v = (0.5 + 0.5 * torch.rand(half, hkv, page, D, generator=g)).to(BF)
    k, v = torch.cat([k, k]).cuda(), torch.cat([v, -v]).cuda()
    table = torch.arange(2 * half, dtype=torch.int32, device="cuda").expand(B, -1)
    q = (torch.randn(B, hkv * G * D, generator=g)).to(BF).cuda()
    n = torch.full((B,), rows, dtype=torch.int32, device="cuda")
    out = ops.paged_attention(q, k, v, table, n, hkv * G, hkv, D).double()
    ops.status_fetch()
    assert float(out.abs().max()) <= 2.0 ** (-19 if G <= 8 else -13), float(out.abs().max())
    assert G > 8 or abs(float(out.mean())) <= 2.0 ** -23, float(out.mean())
