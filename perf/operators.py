"""The decode step of a server whose sequences have lengths of their own, operator by operator.

  attend   one query per sequence over a paged cache (rows of a sequence lie in pages that a table names)
  step     the same behind a projection: queries and keys are normalised and rotated at each sequence's position, the new row
           goes into its page, attention covers it too
  evict    a paged cache is cut back to `keep` rows per sequence and key head: the newest `recent` and those that attention has
           weighed most; the rows behind `keep` that stay move into the places given up in front of it
  sample   the next token of every sequence by temperature, top-k, top-p and min-p, from given uniform numbers

"attend" and "step" add every row's attention weight to an accumulator where the case says so; it is what "evict" goes by.
Head counts and sizes are those of ComplexityConfig's presets, and a few that other groupings need; vocabularies of 32 000
(the bench's) and 100 000 (the presets').
"""
from __future__ import annotations

import math
import random

import torch

own = False

EPS = 1e-6
NEXT = 500            # a sequence that has lost rows stands further along than its number of rows says


def _attn(name, kind, batch, hkv, group, dim, page, longest, weights=False, spread=16, empty=0, order="heads", salt=1):
    """Lengths between longest / spread and longest, and `empty` sequences of none; order: what lies next to one another in a
    page, the rows of a head ("heads") or the heads of a row ("rows")."""
    return {"name": name, "kind": kind, "batch": batch, "hkv": hkv, "group": group, "dim": dim, "page": page, "longest": longest,
            "weights": weights, "spread": spread, "empty": empty, "order": order, "salt": salt}


def _evict(name, layers, batch, hkv, dim, page, longest, keep, recent, salt=1):
    return {"name": name, "kind": "evict", "layers": layers, "batch": batch, "hkv": hkv, "dim": dim, "page": page,
            "longest": longest, "keep": keep, "recent": recent, "salt": salt}


def _sample(name, batch, vocab, dtype, temperature, top_k, top_p, min_p, mixed=False):
    return {"name": name, "kind": "sample", "batch": batch, "vocab": vocab, "dtype": dtype, "temperature": temperature,
            "top_k": top_k, "top_p": top_p, "min_p": min_p, "mixed": mixed}


def listed():
    return [
        # one user's answer from the 150m preset, 300 tokens in: a call as short as they get
        _attn("step_1x301_g3_d64", "step", 1, 4, 3, 64, 16, 300, spread=1),
        # a server's batch on the 1B preset, ragged, with the accumulator that eviction needs
        _attn("step_32x2048_weights", "step", 32, 8, 2, 128, 64, 2047, weights=True, spread=8),
        # 64 sequences of the 1B preset from 1 000 to 16 000 rows: the largest read
        _attn("attend_64x16384", "attend", 64, 8, 2, 128, 64, 16384, spread=16, salt=3),
        # two long documents: few sequences, the length has to be shared out
        _attn("attend_2x32768", "attend", 2, 8, 2, 128, 128, 32768, spread=1),
        # eight query heads to a key head, pages of 16 rows, a padded batch, odd lengths, heads next to one another
        _attn("attend_24x1999_g8_d64_weights", "attend", 24, 2, 8, 64, 16, 1999, weights=True, spread=64, empty=3, order="rows"),
        # one layer of a small model, a few rows over its budget
        _evict("evict_1x301", 1, 1, 4, 64, 16, 301, 256, 32),
        # four layers of the 1B preset's batch, 256 rows over the budget of 2 048
        _evict("evict_4x32x2304", 4, 32, 8, 128, 64, 2304, 2048, 128),
        # long documents cut to a sixteenth behind their prompt
        _evict("evict_4x32768_to_2048", 1, 4, 8, 128, 128, 32768, 2048, 256),
        # one sequence, the rules that generate() has by default
        _sample("sample_1x32000", 1, 32000, "bf16", 1.0, 50, 0.9, 0.0),
        # a batch over the presets' vocabulary, the same rules
        _sample("sample_32x100000", 32, 100000, "bf16", 0.8, 50, 0.9, 0.0),
        # a nucleus without top-k: everything counts
        _sample("sample_64x100000_nucleus", 64, 100000, "bf16", 1.0, 0, 0.95, 0.0),
        # a large batch of fp32 logits, every request with rules of its own (greedy ones among them)
        _sample("sample_256x32000_f32_mixed", 256, 32000, "f32", 1.0, 0, 1.0, 0.0, mixed=True),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """Batches of 1 to 64 sequences of up to 32 768 rows (1 to 16 query heads a key head, pages of 16 to 256 rows, heads of 64 and
    128); caches of 1 to 4 layers cut to between a sixteenth and all but a few of their rows; 1 to 256 rows of 1 000 to 128 000 logits."""
    kind = rng.choice(["attend", "step", "attend", "step", "evict", "evict", "sample", "sample", "sample"])
    if kind == "sample":
        vocab = _log(rng, 1000, 128000)
        batch = _log(rng, 1, max(1, min(256, 8000000 // vocab)))
        c = _sample("", batch, vocab, rng.choice(["bf16", "f32"]), rng.choice([0.0, 0.5, 0.7, 1.0, 1.0, 1.3]),
                    rng.choice([0, 0, 1, 20, 50, 200, 5000]), rng.choice([1.0, 0.5, 0.9, 0.95]), rng.choice([0.0, 0.0, 0.05, 0.2]),
                    rng.random() < 0.4)
    elif kind == "evict":
        layers, hkv, dim = rng.randint(1, 4), rng.choice([1, 2, 4, 8]), rng.choice([64, 128])
        longest = _log(rng, 40, 32768)
        batch = _log(rng, 1, max(1, min(64, 2000000 // (longest * layers * hkv))))
        keep = max(1, min(longest - rng.randint(1, 40), int(longest * rng.choice([0.0625, 0.25, 0.5, 0.9, 1.0]))))
        c = _evict("", layers, batch, hkv, dim, rng.choice([16, 32, 64, 128, 256]), longest, keep, rng.randint(0, keep // 2),
                   rng.randint(1, 10 ** 6))
    else:
        hkv, dim = rng.choice([1, 2, 3, 4, 8]), rng.choice([64, 128])
        group = rng.choice([1, 2, 2, 3, 4, 7, 8, 16])
        longest = _log(rng, 1, 32767)
        batch = _log(rng, 1, max(1, min(64, (1000000 if kind == "attend" else 500000) // (longest * hkv))))
        c = _attn("", kind, batch, hkv, group, dim, rng.choice([16, 32, 64, 128, 256]), longest, rng.random() < 0.5,
                  rng.choice([1, 4, 64]), rng.randint(0, batch // 4), rng.choice(["heads", "rows"]), rng.randint(1, 10 ** 6))
    del c["name"]
    return c


def _lengths(case):
    """Cached rows of each sequence: the longest, then spread evenly over the logarithm, and empty ones last."""
    rng = random.Random(case["salt"])
    if case["kind"] == "evict":                  # behind the same budget all but a few have grown alike
        return [case["longest"] - (rng.randint(0, case["longest"] // 16) if b % 8 == 7 else 0) for b in range(case["batch"])]
    low = max(1, case["longest"] // case["spread"])
    full = [case["longest"]] + [_log(rng, low, case["longest"]) for _ in range(case["batch"] - 1 - case["empty"])]
    return full + [0] * case["empty"]


def _pages(g, case, layers, width):
    """Pools of keys and values with every page in use at a random place, and the table of who has which."""
    batch, hkv, page, dim = case["batch"], case["hkv"], case["page"], case["dim"]
    count = batch * width + 3                                                # a few pages are nobody's
    shape = (layers, count, hkv, page, dim)
    rows = case.get("order") == "rows"
    pools = []
    for _ in range(2):
        at = (layers, count, page, hkv, dim) if rows else shape
        pool = torch.empty(at, dtype=torch.bfloat16, device="cuda").normal_(generator=g)
        pools.append(pool.transpose(2, 3) if rows else pool)
    table = torch.randperm(count, generator=g, device="cuda")[: batch * width].to(torch.int32).view(batch, width)
    return pools[0], pools[1], table


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(7919 * int(seed) + 13)

    def normal(*shape):
        return torch.empty(shape, device="cuda").normal_(generator=g)

    s = {"case": case}
    if case["kind"] == "sample":
        batch, vocab = case["batch"], case["vocab"]
        # a trained model's logits: a wide bulk and a few tokens that stand out
        x = 2.0 * normal(batch, vocab)
        x.scatter_(1, torch.randint(0, vocab, (batch, 20), generator=g, device="cuda"), 6.0 + 2.0 * normal(batch, 20))
        s["logits"] = x.to(torch.bfloat16 if case["dtype"] == "bf16" else torch.float32)
        s["uniform"] = torch.rand(batch, generator=g, device="cuda")
        if case["mixed"]:                        # as requests bring them: a tensor of each
            pick = lambda v, t: torch.tensor(v, dtype=t, device="cuda")[  # noqa: E731
                torch.randint(0, len(v), (batch,), generator=g, device="cuda")]
            s["temperature"] = pick([0.0, 0.6, 0.8, 1.0, 1.2], torch.float32)
            s["top_k"] = pick([0, 1, 40, 50, 1000], torch.int32)
            s["top_p"] = pick([0.8, 0.9, 0.95, 1.0], torch.float32)
            s["min_p"] = pick([0.0, 0.0, 0.02, 0.1], torch.float32)
        else:
            s.update({k: case[k] for k in ("temperature", "top_k", "top_p", "min_p")})
        return s

    lens = _lengths(case)
    batch, hkv, page, dim = case["batch"], case["hkv"], case["page"], case["dim"]
    width = -(-(max(lens) + 1) // page)
    layers = case.get("layers", 1)
    k, v, s["table"] = _pages(g, case, layers, width)
    s["lengths"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
    s["positions"] = s["lengths"] + NEXT
    rows = width * page
    if case["kind"] == "evict":
        s["k"], s["v"] = k, v
        # the weight that hundreds of steps leave on a row: few rows have most of it
        s["weights"] = torch.exp(1.5 * normal(layers, batch, hkv, rows))
        # the newest rows in order behind `keep`, older ones in front in the order that earlier cuts have left
        at = torch.arange(rows, device="cuda").expand(layers, batch, hkv, rows)
        older = torch.rand(layers, batch, hkv, case["keep"], generator=g, device="cuda").argsort(-1)
        s["row_positions"] = (torch.cat([older, at[..., case["keep"]:]], -1) + NEXT).to(torch.int32)
        s["weights_out"] = torch.zeros_like(s["weights"])
        s["row_positions_out"] = torch.zeros_like(s["row_positions"])
        return s
    s["k"], s["v"] = k[0], v[0]
    hq = hkv * case["group"]
    s["qkv"] = normal(batch, (hq + 2 * hkv) * dim).to(torch.bfloat16)
    s["weights"] = torch.exp(normal(batch, hkv, rows)) if case["weights"] else None
    s["row_positions"] = None
    if case["kind"] == "step":
        s["q_w"], s["k_w"] = ((1 + 0.2 * normal(dim)).to(torch.bfloat16) for _ in range(2))
        freq = 1e4 ** (-torch.arange(0, dim, 2, device="cuda", dtype=torch.float64) / dim)
        angle = torch.arange(rows + NEXT + 1, device="cuda", dtype=torch.float64)[:, None] * torch.cat([freq, freq])
        s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
        if case["weights"]:
            s["row_positions"] = torch.zeros(batch, hkv, rows, dtype=torch.int32, device="cuda")
    return s


# --------------------------------------------------------------------------------------- plain forms
def _dense(pages, table):
    """[B, hkv, rows, D] in 32 bits of a pool [P, hkv, page, D]."""
    t = pages[table.long()].float()                                          # [B, width, hkv, page, D]
    return t.permute(0, 2, 1, 3, 4).flatten(2, 3)


def _attend(q, k_pages, v_pages, table, lengths, weights, new):
    """q [B, hkv, G, D] in 32 bits; `new`: the row whose weight is set, where there is one."""
    k, v = _dense(k_pages, table), _dense(v_pages, table)
    at = torch.arange(k.shape[2], device=q.device)
    seen = at < lengths[:, None]                                             # [B, rows]
    score = (q @ k.transpose(2, 3)) * q.shape[-1] ** -0.5
    score = torch.where(seen[:, None, None], score, -torch.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(torch.isfinite(top), top, 0.0))
    total = p.sum(-1, keepdim=True)
    p = torch.where(total > 0, p / total, 0.0)
    out = (p @ torch.where(seen[:, None, :, None], v, 0.0)).flatten(1).to(torch.bfloat16)
    if weights is not None:
        share = p.sum(2)
        fresh = (at == new[:, None])[:, None] if new is not None else torch.zeros_like(seen)[:, None]
        weights.copy_(torch.where(seen[:, None], torch.where(fresh, 0.0, weights) + share, weights))
    return out


def _rotated(x, w, cos, sin):
    """Heads [B, heads, D] in 32 bits: RMS norm with weight, then rotation of the two halves."""
    x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * w.float()
    a, b = x.chunk(2, -1)
    return x * cos[:, None] + torch.cat([-b, a], -1) * sin[:, None]


def _run_step(s):
    c = s["case"]
    hkv, group, dim, page = c["hkv"], c["group"], c["dim"], c["page"]
    batch, hq = c["batch"], hkv * group
    x = s["qkv"].float().view(batch, hq + 2 * hkv, dim)
    at = s["positions"].long()
    cos, sin = s["cos"][at], s["sin"][at]
    q = _rotated(x[:, :hq], s["q_w"], cos, sin).view(batch, hkv, group, dim)
    row = s["lengths"].long()
    where = s["table"].gather(1, (row // page)[:, None])[:, 0].long()
    s["k"][where, :, row % page] = _rotated(x[:, hq:hq + hkv], s["k_w"], cos, sin).to(torch.bfloat16)
    s["v"][where, :, row % page] = s["qkv"].view(batch, hq + 2 * hkv, dim)[:, hq + hkv:]
    if s["row_positions"] is not None:
        s["row_positions"].scatter_(2, row[:, None, None].expand(-1, hkv, 1), s["positions"][:, None, None].expand(-1, hkv, 1))
    return _attend(q, s["k"], s["v"], s["table"], s["lengths"] + 1, s["weights"], s["lengths"])


def _run_evict(s):
    c = s["case"]
    keep, page = c["keep"], c["page"]
    n = s["lengths"][:, None, None]                                          # [B, 1, 1]
    at = torch.arange(s["weights"].shape[-1], device="cuda")
    newest = s["row_positions"] >= s["positions"][:, None, None] - c["recent"]
    key = torch.where(newest, torch.inf, s["weights"])
    key = torch.where(at < n, key, -torch.inf)
    first = torch.sort(key, dim=-1, descending=True, stable=True).indices[..., :keep]
    stays = torch.zeros_like(key, dtype=torch.bool).scatter_(-1, first, True) & (at < n)
    full = n > keep
    holes = torch.nonzero(~stays & (at < keep) & full)                       # [m, 4]: layer, sequence, head, row
    moved = torch.nonzero(stays & (at >= keep) & full)
    layer, b, h, to = holes.unbind(1)
    src = moved[:, 3]
    for_page = lambda r: s["table"][b, r // page].long()  # noqa: E731
    s["k"][layer, for_page(to), h, to % page] = s["k"][layer, for_page(src), h, src % page]
    s["v"][layer, for_page(to), h, to % page] = s["v"][layer, for_page(src), h, src % page]
    held = at < n.clamp(max=keep)
    for name in ("weights", "row_positions"):
        value, out = s[name], s[name + "_out"]
        out.copy_(torch.where(held, value, out))
        out[layer, b, h, to] = value[layer, b, h, src]
    return {"k": s["k"], "v": s["v"], "weights": s["weights_out"], "row_positions": s["row_positions_out"]}


def _column(v, dtype, like):
    t = v if isinstance(v, torch.Tensor) else torch.full((like.shape[0],), v, dtype=dtype, device=like.device)
    return t[:, None]


def _run_sample(s):
    x = s["logits"].double()
    batch, vocab = x.shape
    temperature = _column(s["temperature"], torch.float32, x).double()
    top_k = _column(s["top_k"], torch.int32, x).long()
    top_p = _column(s["top_p"], torch.float32, x).double()
    min_p = _column(s["min_p"], torch.float32, x).double()
    ordered, order = torch.sort(x, dim=-1, descending=True, stable=True)
    best = ordered[:, :1]
    w = torch.exp((ordered - best) / torch.where(temperature > 0, temperature, 1.0))
    place = torch.arange(vocab, device="cuda")
    w = torch.where((temperature > 0) | (place == 0), w, 0.0)
    kth = ordered.gather(1, top_k.clamp(1, vocab) - 1)
    w = torch.where((top_k <= 0) | (ordered >= kth), w, 0.0)
    ahead = torch.cumsum(w, -1) - w
    kept = (top_p >= 1) | (ahead <= top_p * w.sum(-1, keepdim=True))
    kept = kept & (w >= min_p)
    w = torch.zeros_like(w).scatter_(1, order, torch.where(kept, w, 0.0))
    mass = torch.cumsum(w, -1)
    total = mass[:, -1:]
    ids = torch.searchsorted(mass, s["uniform"].double()[:, None] * total, right=True).clamp(max=vocab - 1)
    return ids[:, 0], (w.gather(1, ids) / total)[:, 0].float()


def run(s):
    c = s["case"]
    if own:
        from complexity_deep_b200 import ops
        if c["kind"] == "sample":
            return ops.sample_tokens(s["logits"], s["uniform"], s["temperature"], s["top_k"], s["top_p"], s["min_p"])
        if c["kind"] == "evict":
            ops.evict_rows_(s["k"], s["v"], s["table"], s["lengths"], s["positions"], s["weights"], s["row_positions"], c["keep"],
                            c["recent"], weights_out=s["weights_out"], row_positions_out=s["row_positions_out"])
            return {"k": s["k"], "v": s["v"], "weights": s["weights_out"], "row_positions": s["row_positions_out"]}
        hq = c["hkv"] * c["group"]
        if c["kind"] == "attend":
            out = ops.paged_attention(s["qkv"], s["k"], s["v"], s["table"], s["lengths"], hq, c["hkv"], c["dim"], weights=s["weights"])
        else:
            out = ops.paged_step_attention(s["qkv"], s["q_w"], s["k_w"], s["cos"], s["sin"], EPS, hq, c["hkv"], c["dim"], s["k"], s["v"],
                                           s["table"], s["lengths"], s["positions"], weights=s["weights"],
                                           row_positions=s["row_positions"])
    elif c["kind"] == "sample":
        return _run_sample(s)
    elif c["kind"] == "evict":
        return _run_evict(s)
    elif c["kind"] == "attend":
        q = s["qkv"][:, : c["hkv"] * c["group"] * c["dim"]].float().view(c["batch"], c["hkv"], c["group"], c["dim"])
        out = _attend(q, s["k"], s["v"], s["table"], s["lengths"], s["weights"], None)
    else:
        out = _run_step(s)
    result = {"out": out}
    if s["weights"] is not None:
        result["weights"] = s["weights"]
    if c["kind"] == "step":
        result["k"], result["v"] = s["k"], s["v"]
        if s["row_positions"] is not None:
            result["row_positions"] = s["row_positions"]
    return result


def work(case):
    """Each cached row of keys and values once, each logit once; an eviction reads what it chooses by and moves, of the rows behind
    `keep`, the newest and that share of the others that stays."""
    if case["kind"] == "sample":
        n = case["batch"] * case["vocab"]
        return {"bytes": n * (2 if case["dtype"] == "bf16" else 4) + 28 * case["batch"], "flops": 4 * n}
    lens = _lengths(case)
    hkv, dim = case["hkv"], case["dim"]
    if case["kind"] == "evict":
        keep, recent, moved, seen, left = case["keep"], case["recent"], 0.0, 0, 0
        for n in lens:
            seen += n
            left += min(n, keep)
            if n > keep:
                others = max(0, n - keep - recent)
                moved += n - keep - others + others * (keep - recent) / max(1, n - recent)
        pairs = case["layers"] * hkv
        return {"bytes": int(pairs * (8 * seen + 8 * left + 8 * dim * moved)), "flops": pairs * seen}
    step = case["kind"] == "step"
    rows = sum(lens) + (case["batch"] if step else 0)
    hq = hkv * case["group"]
    a_row = 4 * dim + (8 if case["weights"] else 0)
    io = case["batch"] * dim * 2 * (2 * hq + (4 * hkv if step else 0))
    return {"bytes": rows * hkv * a_row + io, "flops": 4 * hq * dim * rows}


# --------------------------------------------------------------------------------------- in 64 bits
def _exact_sample(s):
    x = s["logits"].double()
    uniform = s["uniform"].double().tolist()
    values = []
    for name in ("temperature", "top_k", "top_p", "min_p"):
        v = s[name]
        if not isinstance(v, torch.Tensor):
            v = torch.full((x.shape[0],), v, dtype=torch.int32 if name == "top_k" else torch.float32)
        values.append(v.double().tolist())
    ids, probs = [], []
    for i, (t, k, p, m) in enumerate(zip(*values)):
        row = x[i]
        if t == 0:
            ids.append(int((row == row.max()).nonzero()[0, 0]))
            probs.append(1.0)
            continue
        w = torch.softmax(row / t, 0)
        if k > 0:
            w = torch.where(row >= row.topk(min(int(k), row.numel())).values[-1], w, 0.0)
        w = w / w.sum()
        if p < 1:
            down, index = torch.sort(w, descending=True, stable=True)
            ahead = torch.cat([down.new_zeros(1), down.cumsum(0)[:-1]])
            w = w.index_fill(0, index[ahead > p], 0.0)
        w = torch.where(row - row.max() >= t * math.log(m), w, 0.0) if m > 0 else w
        w = w / w.sum()
        chosen = min(int((w.cumsum(0) <= uniform[i]).sum()), row.numel() - 1)
        ids.append(chosen)
        probs.append(float(w[chosen]))
    return torch.tensor(ids, device=x.device), torch.tensor(probs, dtype=torch.float64, device=x.device)


def _exact_evict(s):
    c = s["case"]
    keep, page = c["keep"], c["page"]
    k, v, w_out, p_out = s["k"].clone(), s["v"].clone(), s["weights_out"].double(), s["row_positions_out"].clone()
    flat = torch.arange(s["weights"].shape[-1], device="cuda")
    for layer in range(c["layers"]):
        for b, n in enumerate(_lengths(c)):
            limit = n + NEXT - c["recent"]
            for h in range(c["hkv"]):
                w, pos = s["weights"][layer, b, h, :n].double(), s["row_positions"][layer, b, h, :n]
                take = flat[: min(n, keep)].clone()
                if n > keep:
                    rank = torch.argsort(torch.where(pos >= limit, torch.inf, w), descending=True, stable=True)[:keep]
                    lost = torch.ones(n, dtype=torch.bool, device="cuda")
                    lost[rank] = False
                    take[lost[:keep]] = flat[keep:n][~lost[keep:]]
                w_out[layer, b, h, : take.numel()] = w[take]
                p_out[layer, b, h, : take.numel()] = pos[take]
                to = flat[: take.numel()]
                place = s["table"][b].long()
                for pool, source in ((k, s["k"]), (v, s["v"])):
                    pool[layer, place[to // page], h, to % page] = source[layer, place[take // page], h, take % page]
    return {"k": k, "v": v, "weights": w_out, "row_positions": p_out}


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "sample":
        return _exact_sample(s)
    if case["kind"] == "evict":
        return _exact_evict(s)
    hkv, group, dim, page = case["hkv"], case["group"], case["dim"], case["page"]
    hq, step = hkv * group, case["kind"] == "step"
    k, v = s["k"].clone() if step else s["k"], s["v"].clone() if step else s["v"]
    weights = s["weights"].double() if case["weights"] else None
    out = torch.zeros(case["batch"], hkv, group, dim, dtype=torch.float64, device="cuda")
    for b, n in enumerate(_lengths(case)):
        place = s["table"][b].long()
        heads = s["qkv"][b].double().view(hq + 2 * hkv, dim)
        q = heads[:hq]
        if step:
            turned = []
            for x, w in ((heads[:hq], s["q_w"]), (heads[hq:hq + hkv], s["k_w"])):
                x = x / (x.square().mean(1, keepdim=True) + EPS).sqrt() * w.double()
                swapped = torch.cat([-x[:, dim // 2:], x[:, : dim // 2]], 1)
                turned.append(x * s["cos"][n + NEXT].double() + swapped * s["sin"][n + NEXT].double())
            q = turned[0]
            k[place[n // page], :, n % page] = turned[1].float().to(torch.bfloat16)
            v[place[n // page], :, n % page] = s["qkv"][b].view(-1, dim)[hq + hkv:]
            if weights is not None:
                weights[b, :, n] = 0
                s["row_positions"][b, :, n] = n + NEXT
            n += 1
        if n == 0:
            continue
        kk, vv = (t[place[: -(-n // page)]].transpose(0, 1).flatten(1, 2)[:, :n].double() for t in (k, v))
        p = torch.softmax(torch.einsum("hgd,hnd->hgn", q.view(hkv, group, dim), kk) / math.sqrt(dim), -1)
        out[b] = torch.einsum("hgn,hnd->hgd", p, vv)
        if weights is not None:
            weights[b, :, :n] += p.sum(1)
    result = {"out": out.flatten(1)}
    if weights is not None:
        result["weights"] = weights
    if step:
        result["k"], result["v"] = k, v
        if s["row_positions"] is not None:
            result["row_positions"] = s["row_positions"]
    return result
