"""What quantize_projections and add_adapters refuse, they refuse before anything is replaced, in a layer and in a stack; names
may come from any iterable."""

from __future__ import annotations

import pytest
import torch

from common import RELEASE_TOY, model_args
from test_mx8_adapters import ALL, BF, in_8_bits, layer


def stack():
    from dsv41.model import AttentionStack
    return AttentionStack(model_args(RELEASE_TOY), BF, "cpu")


@pytest.fixture
def quantized(monkeypatch):
    """from_linear on the host, by name of what it was given."""
    from dsv41 import mx8
    calls = []

    def from_linear(lin):
        calls.append(lin)
        return in_8_bits(lin)

    monkeypatch.setattr(mx8.MX8Linear, "from_linear", from_linear)
    return calls


def test_a_layer_before_it_replaces_anything(quantized):
    a = layer()
    a.wo_b = torch.nn.Linear(48, a.dim, bias=False, dtype=BF)
    with pytest.raises(ValueError, match="48 channels"):
        a.quantize_projections()
    assert not quantized and not any(type(getattr(a, n)) is not torch.nn.Linear for n in ALL)
    assert set(a.quantize_projections(("wq_a", "wq_b"))) == {"wq_a", "wq_b"}


def test_a_stack_before_its_first_layer(quantized):
    s = stack()
    s.layers[-1].add_adapters(2, 8, ("wkv",))
    with pytest.raises(ValueError, match="wkv has adapters"):
        s.quantize_projections()
    assert not quantized
    s = stack()
    s.layers[-1].quantize_projections(("wkv",))
    with pytest.raises(ValueError, match="wkv is held in 8 bits"):
        s.add_adapters(2, 8)
    assert not any(a.adapters for a in s.layers)


def test_names_from_a_generator(quantized):
    a = layer()
    assert set(a.quantize_projections(n for n in ("wq_a", "wkv"))) == {"wq_a", "wkv"} and len(quantized) == 2
    assert set(a.add_adapters(2, 8, (n for n in ("wq_b", "wo_b")))) == {"wq_b", "wo_b"}
    s = stack()
    assert all(set(d) == {"wq_a", "wkv"} for d in s.quantize_projections(n for n in ("wq_a", "wkv")))
    assert all(set(d) == {"wo_b"} for d in s.add_adapters(2, 8, (n for n in ("wo_b",))))
