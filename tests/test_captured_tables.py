"""What a captured launch reads stays where it is: rotation tables handed out during a capture outlive the longer ones that
take their place (on the CPU, with the state of the stream made up)."""
import gc
import weakref

import torch

from complexity_deep_b200.core import rotary


def _grow(monkeypatch, capturing):
    rot = rotary.RotaryEmbedding(16, max_seq_len=8)
    monkeypatch.setattr(rotary, "_capturing", lambda t: capturing, raising=False)
    rot.tables_fp32(8)
    first = [weakref.ref(t) for t in rot.tables_fp32(8)]
    values, address = rot.cos_cached.clone(), rot.cos_cached.data_ptr()
    monkeypatch.setattr(rotary, "_capturing", lambda t: False, raising=False)
    rot.tables_fp32(100)
    rot.forward(300)
    gc.collect()
    return rot, first, values, address


def test_captured_tables_stay(monkeypatch):
    rot, first, values, address = _grow(monkeypatch, True)
    assert all(t() is not None for t in first)
    assert first[0]().data_ptr() == address and torch.equal(first[0](), values)
    # a cast of the module (which gives it tables of another type) leaves them alone, as does what a checkpoint holds
    rot.to(torch.bfloat16)
    rot.tables_fp32(8)
    gc.collect()
    assert first[0]().dtype is torch.float32 and torch.equal(first[0](), values) and list(rot.state_dict()) == ["inv_freq"]


def test_other_tables_go(monkeypatch):
    assert all(t() is None for t in _grow(monkeypatch, False)[1])


def test_nothing_is_captured_on_the_cpu():
    assert not rotary._capturing(torch.zeros(1))
