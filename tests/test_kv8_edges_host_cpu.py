"""What the cache in 8 bits and its attention refuse beside what test_kv8_host_cpu.py holds: without a GPU."""

import pytest
import torch
from torch.autograd import forward_ad

from dia_tts_prune_b200 import lm_ops
from test_kv8_host_cpu import operands


def test_sinks_with_gradients_and_tangents_are_refused(monkeypatch):
    """Sinks are parameters of trained models: an operator without a gradient says so instead of dropping it."""
    c, q, k, v, table, past, first = operands()
    reached = []
    monkeypatch.setattr(lm_ops, "_check_device", lambda *a: None)
    monkeypatch.setattr(lm_ops, "_call", lambda what, *a: reached.append(what))
    sinks = torch.nn.Parameter(torch.zeros(4))
    with pytest.raises(ValueError, match="gradient"):
        lm_ops.attention_kv8(q, c, table, past, first, sinks=sinks)
    with pytest.raises(ValueError, match="gradient"):
        lm_ops.attention_kv8(q, c, table, past, first, sinks=2 * sinks)
    with forward_ad.dual_level():
        with pytest.raises(ValueError, match="tangent"):
            lm_ops.attention_kv8(q, c, table, past, first, sinks=forward_ad.make_dual(torch.zeros(4), torch.ones(4)))
    assert not reached
    with torch.no_grad():
        lm_ops.attention_kv8(q, c, table, past, first, sinks=sinks)
    lm_ops.attention_kv8(q, c, table, past, first, sinks=sinks.detach())
    assert reached == ["kv8_attention"] * 2
