"""GELU in the products' epilogue over its whole left tail, with a relative bound.

erfc(a / sqrt 2) / 2 = q(a) exp(-a^2 / 2): the formula for q is within 4.11e-6 = 69 * 2^-24 of it, relatively. In steps of
2^-24: t = 1 / (1 + 0.3085 a) is 3 off (a product's and a reciprocal's step), and q's relative change is at most 3 times t's;
the six multiply-adds 8, the products with exp and v 3, the exponential itself 4, and its argument -v^2/2 one step of its own, one
of the product with log2 e and half a one of that constant: 1.25 v^2. Sum 93 + 1.25 v^2; 96 + 2 v^2 is asked for, and half a
bf16 step for the rounding. Results under the smallest normal value, 2^-126, may be anything under it."""

from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows", [1, 70])
@pytest.mark.parametrize("odd", [0, 1])
def test_gelu_keeps_its_relative_error(gpu, rows, odd):
    """Products of zeros, so that the bias is what is activated, in rows that are aligned and not."""
    from dsv41 import mx8
    v = torch.cat([torch.linspace(-13.5, 9.0, 45000), -torch.logspace(-30, 1.12, 4000), torch.logspace(-30, 30, 3000),
                   torch.tensor([0.0, -0.0, math.inf, -100.0, -3e38] + [0.0] * 3)])
    v = v[odd:]
    n = v.numel()
    assert (n % 8 != 0) == bool(odd)
    w = mx8.Quantized(torch.zeros(n, 64, dtype=torch.uint8, device=gpu), torch.full((n, 2), 127, dtype=torch.uint8, device=gpu))
    x = mx8.Quantized(torch.zeros(rows, 64, dtype=torch.uint8, device=gpu), torch.full((rows, 2), 127, dtype=torch.uint8, device=gpu))
    got = mx8.MX8Linear(*w, v.to(gpu))(x, activation="gelu").double().cpu()
    d = v.double()
    want = 0.5 * d * torch.special.erfc(-d * math.sqrt(0.5))
    fine = want.isfinite()
    assert (got[:, ~fine] == want[~fine]).all()
    size, steps = want[fine].abs(), (96 + 2 * d[fine].square().clamp(max=400.0)) * 2.0 ** -24
    near = size * (2.0 ** -8 * (1 + steps) + steps) + (size < 2.0 ** -126) * 2.0 ** -126
    off = (got[:, fine] - want[fine]).abs()
    assert (off <= near).all(), (d[fine][(off > near)[0]][:8], (off / size)[off > near][:8])
