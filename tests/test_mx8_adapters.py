"""Projections in 8 bits and adapters on one projection are refused in whatever order they come, on the host."""

from __future__ import annotations

import pytest
import torch

from common import C1, RELEASE_TOY, model_args

BF, U8 = torch.bfloat16, torch.uint8
ALL = ("wq_a", "wkv", "wq_b", "wo_b")


def layer(cfg=RELEASE_TOY, dtype=BF):
    from dsv41.attention import Attention
    return Attention(0, model_args(cfg), dtype, "cpu")


def in_8_bits(lin):
    from dsv41.mx8 import MX8Linear
    n, k = lin.weight.shape
    return MX8Linear(torch.zeros(n, k, dtype=U8), torch.zeros(-(-n // 32), k // 32, dtype=U8))


@pytest.mark.parametrize("name", ALL)
def test_assigned_where_adapters_are(name):
    a = layer()
    a.add_adapters(2, 8)
    held = getattr(a, name)
    with pytest.raises(ValueError, match=f"{name} has adapters"):
        setattr(a, name, in_8_bits(held))
    assert getattr(a, name) is held
    del a.adapters[name]
    setattr(a, name, in_8_bits(held))
    assert getattr(a, name) is not held


@pytest.mark.parametrize("name", ALL)
def test_a_bank_put_beside_a_projection_in_8_bits(name):
    """A bank that did not come through add_adapters, and a projection that did not come as an attribute."""
    from dsv41.adapters import AdapterBank
    from dsv41.model import SharedState
    for first in ("projection", "bank"):
        a = layer()
        n, k = getattr(a, name).weight.shape
        if first == "projection":
            setattr(a, name, in_8_bits(getattr(a, name)))
            a.adapters[name] = AdapterBank(2, k, n, 8, BF, "cpu")
        else:
            a.add_adapters(2, 8, (name,))
            a._modules[name] = in_8_bits(getattr(a, name))
        shared = SharedState()
        shared.adapter_ids = torch.tensor([0], dtype=torch.int32)
        with pytest.raises(ValueError, match=f"{name} is held in 8 bits"):
            a(torch.zeros(1, 1, a.dim, dtype=BF), 0, None, shared)


def test_assigned_to_a_layer_of_another_type():
    a = layer(C1, torch.float32)
    with pytest.raises(ValueError, match="bfloat16"):
        a.wq_b = in_8_bits(a.wq_b)


def test_a_stack_refuses_before_its_first_layer():
    from dsv41.model import AttentionStack
    s = AttentionStack(model_args(RELEASE_TOY), BF, "cpu")
    s.add_adapters(2, 8, ("wo_b",))
    ran = []
    s.layers[0].register_forward_pre_hook(lambda m, args: ran.append(m))
    s.layers[-1]._modules["wo_b"] = in_8_bits(s.layers[-1].wo_b)

    class Cache:
        offset = 0

    with pytest.raises(ValueError, match="wo_b is held in 8 bits"):
        s(torch.zeros(1, 1, s.args.dim, dtype=BF), Cache(), torch.tensor([0], dtype=torch.int32))
    assert not ran
