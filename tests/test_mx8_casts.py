"""An 8-bit projection inside a model whose types are cast keeps what its product takes: uint8 codes and scales, a float32 bias."""

from __future__ import annotations

import pytest
import torch

BF, U8 = torch.bfloat16, torch.uint8


@pytest.mark.parametrize("cast", [lambda m: m.to(BF), lambda m: m.bfloat16(), lambda m: m.half(), lambda m: m.double(),
                                  lambda m: m.to("cpu", BF), lambda m: m.to(BF).float(), lambda m: m.to("meta", BF)])
@pytest.mark.parametrize("bias", [True, False])
def test_a_cast_leaves_the_bias(cast, bias):
    from dsv41 import mx8
    held = torch.randn(40) if bias else None
    m = mx8.MX8Linear(torch.zeros(40, 64, dtype=U8), torch.zeros(2, 2, dtype=U8), held)
    outer = torch.nn.Sequential(torch.nn.Linear(4, 4), m)
    outer = cast(outer)
    assert outer[1] is m and m.codes.dtype == m.scales.dtype == U8
    if not bias:
        assert m.bias is None
    else:
        assert m.bias.dtype == torch.float32 and m.bias.device == m.codes.device == outer[0].weight.device
        if m.bias.device.type != "meta":
            assert torch.equal(m.bias, held)
    assert set(m.state_dict()) == ({"codes", "scales", "bias"} if bias else {"codes", "scales"})
