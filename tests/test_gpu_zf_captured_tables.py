"""Captured steps behind a forward call that is longer than the rotation tables they were captured with: new tables have taken the
old ones' place and other tensors the memory of whatever was given back."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _model(seed=0):
    from complexity_deep_b200.models import ComplexityConfig, ComplexityModel
    torch.manual_seed(seed)
    cfg = ComplexityConfig(vocab_size=500, hidden_size=256, intermediate_size=512, num_hidden_layers=2, num_attention_heads=4,
                           num_key_value_heads=2, num_experts=4, eos_token_id=-1, max_position_embeddings=128)
    return cfg, ComplexityModel(cfg).to("cuda", torch.bfloat16).eval()


def _outgrow(cfg, model):
    """A prompt behind the tables' end, then tensors of the old tables' size and others all over the free memory."""
    before = model.layers[0].self_attn.rotary_emb.cos_cached.shape[0]
    with torch.no_grad():
        model(torch.arange(before + 40, device="cuda")[None] % cfg.vocab_size)
    assert model.layers[0].self_attn.rotary_emb.cos_cached.shape[0] > before
    return [torch.full((n,), float("nan"), device="cuda") for n in [before * 64] * 64 + [64 * 64] * 64]


def test_paged_decoder():
    from complexity_deep_b200.models import PagedDecoder
    cfg, model = _model()
    kw = dict(slots=2, pages=16, page=16, max_rows=100)
    dec, ref = PagedDecoder(model, **kw), PagedDecoder(model, **kw)
    prompt = torch.arange(20) * 7 % cfg.vocab_size
    for d in (dec, ref):
        d.add(prompt, 0.4)
    junk = _outgrow(cfg, model)
    for i in range(6):
        u = torch.full((2,), 0.1 + 0.15 * i, device="cuda")
        ids, probs = dec.step(u)
        ref.cache.reserve()
        ref.uniform.copy_(u)
        with torch.no_grad():
            want = ref._eager_step()
        ref.cache.advance_host()
        assert int(ids[0]) == int(ref.ids[0, 0]) and float(probs[0]) == float(want[0])
    assert torch.equal(dec.cache.k, ref.cache.k) and len(junk) == 128


def test_decode_graph_and_prefill_graph():
    from complexity_deep_b200.models import DecodeGraph, PrefillGraph
    cfg, model = _model(1)
    ids = torch.arange(40, device="cuda").view(2, 20) * 3 % cfg.vocab_size
    dec, pre = DecodeGraph(model, batch=2, capacity=60), PrefillGraph(model, batch=2, seq_len=20)
    dec.prefill(ids)
    want = pre(ids).clone()
    steps = [dec.step(ids[:, i:i + 1]).clone() for i in range(4)]
    junk = _outgrow(cfg, model)
    assert torch.equal(pre(ids), want)
    dec.prefill(ids)
    for i in range(4):
        assert torch.equal(dec.step(ids[:, i:i + 1]), steps[i])
    assert len(junk) == 128
