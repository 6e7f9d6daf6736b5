"""Paged attention holds what is not bf16 to begin with in 32 bits: the weights of rows, and a step's normalised and rotated
queries.  The inputs make the last of those bits the whole result, and everything else about it exact."""
import pytest
import torch

import paged_cases as cases

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def _pieces(x, n):
    """The first n bf16 numbers that x (64 bits) is the sum of, each the nearest to what is left."""
    out = []
    for _ in range(n):
        out.append(float(torch.tensor(x, dtype=torch.float64).to(BF)))
        x -= out[-1]
    return out


def _place(length, rows, seed):
    g = torch.Generator().manual_seed(seed)
    return torch.randperm(length, generator=g)[:rows].tolist()


def _pools(length, D, page, room=0):
    k, v, table = cases.make_cache([length], 1, D, page, 1, rest=0.0, room=room)
    return torch.zeros_like(k), torch.zeros_like(v), table


@pytest.mark.parametrize("G,D", [(1, 64), (8, 64), (2, 128), (16, 64), (9, 128), (16, 128)])
@pytest.mark.parametrize("length", [60, 700, 30000])
def test_weights_of_rows(G, D, length):
    """48 rows of weight w < 1 and value 1, three of weight 1 whose values add up to -48 w: what is left is how w has been rounded.
    Two bf16 numbers are off by up to 2^-17 of w, and this w by more than 2^-18.1.  In 32 bits the score's product with its
    scale (2^-24 of it, twice, of a score of about -1.44 at most: 2^-22.5 of w), exp2 (2 ulp: 2^-22) and the sums (48 additions in
    groups, 2^-24 each of what they hold: below 2^-21.5) stay below 2^-20 together."""
    from complexity_deep_b200 import ops
    scale = float(torch.tensor(D ** -0.5, dtype=torch.float32))

    def left(key):
        w = torch.exp(torch.tensor(-key * scale, dtype=torch.float64)).item()
        return abs(w - sum(_pieces(w, 2))) / w
    key = max((0.5 + i / 16 if D == 64 else 1.0 + i / 8 for i in range(128)), key=lambda c: left(c) if c * scale <= 1.0 else 0.0)
    key = float(torch.tensor(key).to(BF))
    assert left(key) > 2.0 ** -18.1
    w = torch.exp(torch.tensor(-key * scale, dtype=torch.float64)).item()
    k, v, table = _pools(length, D, 16)
    at = _place(length, 51, G + D)
    put = lambda pool, row, x: pool[table[0, row // 16], 0, row % 16].copy_(x)  # noqa: E731
    first = torch.zeros(D, dtype=BF)
    first[0] = 1.0
    for r in range(length):
        put(k, r, first * -2048.0)                                         # no weight at all
    for r in at[:48]:
        put(k, r, first * -key)
        put(v, r, torch.ones(D, dtype=BF))
    for r, part in zip(at[48:], _pieces(48 * w, 3)):
        put(k, r, first * 0.0)
        put(v, r, torch.full((D,), -part, dtype=BF))
    q = first.repeat(G)[None].cuda()
    out = ops.paged_attention(q, k.cuda(), v.cuda(), table.cuda(), torch.tensor([length], dtype=torch.int32, device="cuda"), G, 1, D)
    off = out.double().abs().max().item() * (48 * w + 3) / (48 * w)
    assert off <= 2.0 ** -20, off


@pytest.mark.parametrize("G,D", [(1, 64), (8, 64), (2, 128), (16, 64), (9, 128), (16, 128)])
@pytest.mark.parametrize("lengths", [[3], [700], [30000], [40, 0, 90, 64, 200] * 30])
def test_rotated_queries(G, D, lengths):
    """Queries of 1 + 2^-9 + 2^-20 and 1 + 2^-9 in turn (by the rotation's table; two bf16 numbers hold 1 + 2^-9 of both) against a key of
    +-64 in turn: the score is 32 sqrt(D) 2^-20 and nothing else, 0 where q has 16 bits.  Every sum on the way has at most 21 bits; the weight of that row against one of score 0 is
    exp of it, good to exp2 (2 ulp: 2^-22) and the sum over 16 heads (15 additions: below 2^-20)."""
    from complexity_deep_b200 import ops
    page, hkv = 16, 2
    B, hq = len(lengths), hkv * G
    k, v, table = cases.make_cache(lengths, hkv, D, page, 1, rest=0.0, room=1)
    k, v = torch.zeros_like(k), torch.zeros_like(v)
    turn = torch.tensor([64.0, -64.0] * (D // 2)).to(BF)
    where = [_place(n, 1, n)[0] if n else None for n in lengths]
    for b, r in enumerate(where):
        if r is not None:
            k[table[b, r // page], :, r % page] = turn
    qkv = torch.zeros(B, (hq + 2 * hkv) * D, dtype=BF)
    qkv[:, : hq * D] = 1.0
    cos = torch.full((1, D), 1 + 2.0 ** -9)
    cos[:, ::2] += 2.0 ** -20
    n = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    acc = torch.zeros(B, hkv, table.shape[1] * page, device="cuda")
    ops.paged_step_attention(qkv.cuda(), None, None, cos.cuda(), torch.zeros(1, D, device="cuda"), 0.0, hq, hkv, D, k.cuda(), v.cuda(),
                             table.cuda(), n, torch.zeros(B, dtype=torch.int32, device="cuda"), weights=acc)
    ops.status_fetch()
    score = 32 * 2.0 ** -20 * D * float(torch.tensor(D ** -0.5, dtype=torch.float32))
    acc = acc.double().cpu()
    for b, r in enumerate(where):
        if r is not None:
            ratio = acc[b, :, r] / acc[b, :, lengths[b]]                   # the new row's key is zero
            assert bool(((ratio - torch.exp(torch.tensor(score, dtype=torch.float64))).abs() <= 2.0 ** -18).all()), ratio
