"""Paged caches for tests, and what the operators on them give in 64 bits, sequence by sequence."""
import torch

BF = torch.bfloat16
EPS = 1e-6


def make_cache(lengths, hkv, dim, page, seed, width=None, spare=3, order="heads", room=0, rest=float("nan"), layers=None):
    """Pools with the rows of every sequence at random pages, everything else (rows behind a sequence's end, pages that nobody
    has) filled with `rest`; the table's entries behind a sequence's pages are far outside the pool.  `room`: rows more than
    `lengths` that the table has pages for."""
    g = torch.Generator().manual_seed(seed)
    B = len(lengths)
    need = [-(-max(0, n + room) // page) for n in lengths]
    width = width or max(1, max(need))
    pages = sum(need) + spare
    ids = torch.randperm(pages, generator=g).tolist()
    table = torch.full((B, width), 2 ** 30, dtype=torch.int32)
    lead = (layers,) if layers else ()
    at = lead + ((pages, hkv, page, dim) if order == "heads" else (pages, page, hkv, dim))
    pools = []
    for _ in range(2):
        pool = torch.full(at, rest, dtype=BF)
        pools.append(pool if order == "heads" else pool.transpose(-3, -2))
    for b, n in enumerate(lengths):
        mine = [ids.pop() for _ in range(need[b])]
        table[b, : len(mine)] = torch.tensor(mine, dtype=torch.int32)
        for r in range(0, max(0, n), page):
            m = min(page, n - r)
            for pool in pools:
                pool[..., mine[r // page], :, :m, :] = torch.randn(*lead, hkv, m, dim, generator=g).to(BF)
    return pools[0], pools[1], table


def rows_of(pool, table, b, n):
    """[hkv, n, D] of sequence b in 64 bits."""
    page = pool.shape[2]
    ids = table[b, : -(-n // page)].long()
    return pool[ids].transpose(0, 1).flatten(1, 2)[:, :n].double()


def attend(q, k_pages, v_pages, table, lengths, hkv):
    """q [B, hq, D] in 64 bits -> (out [B, hq, D], sum of p |v| of the same shape, p summed over a head's queries [B][hkv, n])."""
    B, hq, D = q.shape
    out, size, share = torch.zeros(B, hq, D, dtype=torch.float64), torch.zeros(B, hq, D, dtype=torch.float64), []
    for b, n in enumerate(lengths):
        if n <= 0:
            share.append(torch.zeros(hkv, 0, dtype=torch.float64))
            continue
        k, v = rows_of(k_pages, table, b, n), rows_of(v_pages, table, b, n)
        p = torch.softmax(q[b].view(hkv, hq // hkv, D) @ k.transpose(1, 2) * D ** -0.5, -1)
        out[b], size[b] = (p @ v).reshape(hq, D), (p @ v.abs()).reshape(hq, D)
        share.append(p.sum(1))
    return out, size, share


def rotate(x, w, cos, sin):
    """Heads [heads, D] in 64 bits: RMS norm (w or None), rotation of the halves."""
    if w is not None:
        x = x / (x.square().mean(-1, keepdim=True) + EPS).sqrt() * w.double()
    a, b = x.chunk(2, -1)
    return x * cos.double() + torch.cat([-b, a], -1) * sin.double()


def tables(rows, dim):
    freq = 1e4 ** (-torch.arange(0, dim, 2, dtype=torch.float64) / dim)
    angle = torch.arange(rows, dtype=torch.float64)[:, None] * torch.cat([freq, freq])
    return angle.cos().float(), angle.sin().float()


def evict(weights, row_positions, n, limit, keep):
    """Rows that end up at 0 .. keep - 1 of one (sequence, head), by sorting."""
    if n <= keep:
        return list(range(n))

    def rank(i):
        w = weights[i]
        if row_positions[i] >= limit:                 # all alike: only their order in the cache counts
            return 0, 0, 0, i
        return 1, -1 if w != w else 0, -w if w == w else 0, i
    stay = set(sorted(range(n), key=rank)[:keep])
    movers = iter([i for i in range(keep, n) if i in stay])
    return [i if i in stay else next(movers) for i in range(keep)]


def sample(x, u, t, k, p, m):
    """(id, probability) of one row of logits in 64 bits."""
    x = torch.where(x.isnan(), -torch.inf, x.double())
    top = x.max()
    if top == -torch.inf:
        return 0, 0.0
    if not t > 0:
        return int((x == top).nonzero()[0, 0]), 1.0
    w = torch.where(x == top, 1.0, torch.exp(torch.where(x == top, 0.0, x - top) / t))
    w = torch.where(x == -torch.inf, 0.0, w)
    if 0 < k < x.numel():
        w = torch.where(x >= x.sort(descending=True).values[k - 1], w, 0.0)
    if p < 1:
        order = sorted(range(x.numel()), key=lambda i: (-float(x[i]), i))
        ordered = w[order]
        ahead = torch.cumsum(ordered, 0) - ordered
        w[torch.tensor(order)[ahead > max(0.0, p) * ordered.sum()]] = 0.0
    w = torch.where(w >= m, w, 0.0)
    mass = w.cumsum(0)
    i = min(int((mass <= u * mass[-1]).sum()), x.numel() - 1)
    return i, float(w[i] / mass[-1])
