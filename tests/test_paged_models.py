"""Models that the paged operators do not take are refused before a pool is allocated."""
import pytest
import torch

from complexity_deep_b200.models import ComplexityConfig, ComplexityModel
from complexity_deep_b200.models import modeling


def _model(hidden, heads, kv, dtype=torch.bfloat16):
    cfg = ComplexityConfig(vocab_size=32, hidden_size=hidden, intermediate_size=64, num_hidden_layers=1, num_attention_heads=heads,
                           num_key_value_heads=kv, num_experts=2)
    return ComplexityModel(cfg).to(dtype)


@pytest.mark.parametrize("hidden,heads,kv,dtype", [(80, 2, 1, torch.bfloat16), (160, 2, 1, torch.bfloat16), (1088, 17, 1, torch.bfloat16),
                                                   (128, 2, 1, torch.float32)])
def test_refused(monkeypatch, hidden, heads, kv, dtype):
    monkeypatch.setattr(modeling, "PagedKVCache", lambda *a: pytest.fail("a pool has been asked for"))
    with pytest.raises(RuntimeError, match="heads of 64 or 128"):
        _model(hidden, heads, kv, dtype).make_paged_cache(2, 4, 16, 32)


@pytest.mark.parametrize("hidden,heads,kv", [(128, 2, 1), (256, 2, 2), (1024, 16, 1)])
def test_taken(hidden, heads, kv):
    cache = _model(hidden, heads, kv).make_paged_cache(2, 4, 16, 32, statistics=True)
    assert cache.k.shape == (1, 4, kv, 16, hidden // heads) and cache.weights.shape == (1, 2, kv, 32)
