"""Decode steps on a paged cache through the model: sequences of different lengths beside each other against the fp32 oracle and the
contiguous cache, captured steps with sampling and eviction, generate() from given numbers, the command line."""
import pytest
import torch

import paged_cases as cases
from conftest import assert_close

from oracle import complexity_oracle as oracle

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def _model(seed=0, **kw):
    from complexity_deep_b200.models import ComplexityConfig, ComplexityModel
    torch.manual_seed(seed)
    d = dict(vocab_size=500, hidden_size=256, intermediate_size=512, num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=2,
             num_experts=4, eos_token_id=-1)
    d.update(kw)
    cfg = ComplexityConfig(**d)
    return cfg, ComplexityModel(cfg).to("cuda", BF).eval()


def test_steps_against_oracle_and_contiguous_cache():
    from complexity_deep_b200.core.attention import StaticKVCache
    cfg, model = _model()
    g = torch.Generator().manual_seed(1)
    lens, steps = [5, 33, 16], 4
    ids = [torch.randint(0, cfg.vocab_size, (n + steps,), generator=g) for n in lens]
    cache = model.make_paged_cache(slots=4, pages=20, page=16, max_rows=48, statistics=True)
    state = {k: (v.float().cpu() if v.is_floating_point() else v.cpu()) for k, v in model.state_dict().items()}
    with torch.no_grad():
        slots = [cache.add(model(s[None, :n].cuda(), use_cache=True).past_key_values) for s, n in zip(ids, lens)]
        got = []
        for step in range(steps):
            cache.reserve()
            now = torch.zeros(4, 1, dtype=torch.int64)
            for slot, s, n in zip(slots, ids, lens):
                now[slot, 0] = s[n + step]
            got.append(model(now.cuda(), past_key_values=cache.as_past(), use_cache=True).logits.clone())
            cache.advance()
        for slot, s, n in zip(slots, ids, lens):
            ref, _ = oracle.model_forward(state, cfg.to_dict(), s[None])
            alone = StaticKVCache(cfg.num_hidden_layers, 1, 2, 64, n + steps, "cuda")
            alone.load(model(s[None, :n].cuda(), use_cache=True).past_key_values)
            for step in range(steps):
                one = model(s[None, n + step:n + step + 1].cuda(), past_key_values=alone.layers, use_cache=True).logits
                alone.advance()
                assert_close(got[step][slot], ref[0, n + step:n + step + 1], what="oracle")
                assert_close(got[step][slot], one[0].float().cpu(), what="contiguous cache")
            assert cache.length(slot) == n + steps and int(cache.lengths[slot]) == n + steps == int(cache.positions[slot])
            # every step hands out one unit of weight per query head
            total = cache.weights[:, slot].sum(-1)
            assert bool(((total - 2 * steps).abs() < 1e-3).all())
            rows = torch.arange(n + steps, dtype=torch.int32, device="cuda")
            assert bool((cache.row_positions[:, slot, :, : n + steps] == rows).all())
    assert int(cache.lengths[3]) == -1 and int(cache.positions[3]) == 0


@pytest.mark.parametrize("keep", [0, 40])
def test_captured_steps_equal_eager_ones(keep):
    """Prompts that come at different times, rules of their own, a slot that is given back, evictions: the captured step gives
    the tokens, probabilities and caches that the same calls give one by one."""
    from complexity_deep_b200 import ops
    from complexity_deep_b200.models import PagedDecoder
    cfg, model = _model(3)
    g = torch.Generator().manual_seed(2)
    kw = dict(slots=3, pages=12, page=16, max_rows=64, max_positions=200, keep=keep, recent=8 if keep else 0)
    dec, ref = PagedDecoder(model, **kw), PagedDecoder(model, **kw)
    prompts = [torch.randint(0, cfg.vocab_size, (n,), generator=g) for n in (40, 7, 50, 3)]
    rules = [dict(temperature=0.0), dict(temperature=0.8, top_k=20, top_p=0.9), dict(temperature=1.2, top_k=0, min_p=0.02), dict()]
    slots = []
    for d in (dec, ref):
        slots.append([d.add(p, 0.25, **r)[0] for p, r in zip(prompts[:2], rules)])
    for step in range(34 if keep else 20):
        if step == 5:
            for d in (dec, ref):
                d.add(prompts[2], 0.5, **rules[2])
        if step == 9:
            for d, s in zip((dec, ref), slots):
                d.release(s[0])
                d.add(prompts[3], 0.75, **rules[3])
        if not keep and step >= 14:
            break
        u = torch.rand(3, generator=g).cuda()
        ids, probs = dec.step(u)
        if keep and ref.cache.full():
            ref.cache.evict(keep, 8)
        ref.cache.reserve()
        ref.uniform.copy_(u)
        with torch.no_grad():
            want = ref._eager_step()
        ref.cache.advance_host()
        live = [s for s in range(3) if dec.cache.length(s) >= 0]
        assert torch.equal(ids[live], ref.ids[live, 0]) and torch.equal(probs[live], want[live])
        assert torch.equal(dec.cache.lengths, ref.cache.lengths)
        assert dec.cache.lengths.tolist() == [dec.cache.length(s) for s in range(3)]
        if keep:
            assert max(dec.cache.lengths.tolist()) <= 64
    if keep:
        assert torch.equal(dec.cache.weights, ref.cache.weights) and torch.equal(dec.cache.row_positions, ref.cache.row_positions)
        assert torch.equal(dec.cache.k, ref.cache.k) and torch.equal(dec.cache.v, ref.cache.v)


def test_eviction_keeps_what_was_weighed_most():
    """One eviction in the middle of a run, against sorting; the tokens that stay go on being attended at their places."""
    cfg, model = _model(4)
    g = torch.Generator().manual_seed(5)
    prompts = [torch.randint(0, cfg.vocab_size, (n,), generator=g) for n in (60, 30)]
    cache = model.make_paged_cache(2, 10, 16, 80, 200, statistics=True)
    with torch.no_grad():
        for p in prompts:
            cache.add(model(p[None].cuda(), use_cache=True).past_key_values)
        step = lambda: (cache.reserve(), model(torch.ones(2, 1, dtype=torch.int64, device="cuda"), past_key_values=cache.as_past(),  # noqa: E731
                                               use_cache=True), cache.advance())
        for _ in range(10):
            step()
        w, pos, free = cache.weights.cpu(), cache.row_positions.cpu(), cache.free_pages
        before = [cases.rows_of(cache.k[i].cpu(), cache.table.cpu(), 0, 70) for i in range(2)]
        cache.evict(50, 6)
        assert [cache.length(s) for s in range(2)] == cache.lengths.tolist() == [50, 40] and cache.free_pages == free + 1
        for layer in range(2):
            after = cases.rows_of(cache.k[layer].cpu(), cache.table.cpu(), 0, 50)
            for h in range(2):
                src = cases.evict(w[layer, 0, h].tolist(), pos[layer, 0, h].tolist(), 70, 70 - 6, 50)
                assert torch.equal(after[h], before[layer][h][src])
                assert cache.row_positions[layer, 0, h, :50].tolist() == pos[layer, 0, h][src].tolist()
        for _ in range(3):
            step()
        assert cache.lengths.tolist() == [53, 43] and cache.positions.tolist() == [73, 43]
        assert bool((cache.row_positions[:, 0, :, 50:53] == torch.tensor([70, 71, 72], device="cuda")).all())
    from complexity_deep_b200 import ops
    ops.status_fetch()


def test_generate_from_given_numbers():
    cfg, model = _model(6)
    ids = torch.randint(0, cfg.vocab_size, (2, 9), generator=torch.Generator().manual_seed(7)).cuda()
    u = torch.rand(4, 2, generator=torch.Generator().manual_seed(8)).cuda()
    a = model.generate(ids, max_new_tokens=4, temperature=0.9, top_k=30, top_p=0.8, min_p=0.01, uniforms=u)
    b = model.generate(ids, max_new_tokens=4, temperature=0.9, top_k=30, top_p=0.8, min_p=0.01, uniforms=u)
    assert a.shape == (2, 13) and torch.equal(a, b)
    with torch.no_grad():
        first = model(ids).logits[:, -1]
    f32 = lambda v: float(torch.tensor(v))  # noqa: E731
    for row in range(2):
        assert int(a[row, 9]) == cases.sample(first[row].cpu(), float(u[0, row]), f32(0.9), 30, f32(0.8), f32(0.01))[0]
    assert model.generate(ids, max_new_tokens=3, min_p=0.05).shape == (2, 12)
    greedy = model.generate(ids, max_new_tokens=4, do_sample=False)
    assert torch.equal(greedy, model.generate(ids, max_new_tokens=4, do_sample=False, uniforms=u))


def test_paged_generate_and_command_line(tmp_path, capsys):
    from complexity_deep_b200 import cli
    from complexity_deep_b200.models import paged_generate
    cfg, model = _model(9)
    prompts = [[3, 5, 7, 11, 13], [2], list(range(40))]
    a = paged_generate(model, prompts, 20, 0.8, 20, 0.9, page=16, seed=1)
    assert a == paged_generate(model, prompts, 20, 0.8, 20, 0.9, page=16, seed=1)
    assert [len(x) for x in a] == [25, 21, 60] and [x[: len(p)] for x, p in zip(a, prompts)] == prompts
    cut = paged_generate(model, prompts, 20, 0.8, 20, 0.9, page=16, keep=24, recent=4, seed=1)
    assert [len(x) for x in cut] == [25, 21, 60]
    eos = a[0][7]
    stopped = paged_generate(model, prompts, 20, 0.8, 20, 0.9, page=16, seed=1, eos_token_id=eos)
    assert stopped[0][-1] == eos and stopped[0] == a[0][: len(stopped[0])]
    model.save_pretrained(str(tmp_path))
    args = [x for p in prompts for x in ("--prompt", ",".join(map(str, p)))]
    assert cli.main(["generate", "--model", str(tmp_path), "--paged", "--page-size", "16", "--seed", "1", "--temperature", "0.8", "--top-k",
                     "20", "--max-new-tokens", "20"] + args) == 0
    assert [list(map(int, line.split(","))) for line in capsys.readouterr().out.split()] == a


def test_refusals():
    from complexity_deep_b200.models import PagedDecoder
    cfg, model = _model(10)
    with pytest.raises(ValueError):
        PagedDecoder(model, 1, 4, 16, 32, keep=32)
    dec = PagedDecoder(model, slots=1, pages=2, page=16, max_rows=64)
    dec.add(torch.arange(32))
    with pytest.raises(RuntimeError, match="no page left"):
        dec.step(torch.zeros(1, device="cuda"))
    with pytest.raises(RuntimeError, match="slots"):
        dec.add(torch.arange(3))
    with torch.no_grad(), pytest.raises(RuntimeError, match="one new token per slot"):
        model(torch.zeros(2, 1, dtype=torch.int64, device="cuda"), past_key_values=dec.cache.as_past(), use_cache=True)
