"""SiLU in the products' epilogue down to the smallest normal result, with a relative bound.

v 2^-8 / (2^-8 + 2^-8 exp(-v)), in steps of 2^-24 of the result: the exponential's argument -8 - v log2 e is rounded once, at most
8 + 1.45 |v| of them (times log 2 in the result: 6 + |v|), and its constant half a |v|; the exponential itself 4, the sum 1, the
reciprocal 2, the products 3. Sum 16 + 1.5 |v|; 32 + 2 |v| is asked for, and half a bf16 step for the rounding. Where v 2^-8 is no
normal number its rounding, 2^-150, comes to 2^-142 in the result. Results under the smallest normal value, 2^-126, may be anything
under it."""

from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows", [1, 70])
@pytest.mark.parametrize("odd", [0, 1])
def test_silu_keeps_its_relative_error(gpu, rows, odd):
    """Products of zeros, so that the bias is what is activated, in rows that are aligned and not."""
    from dsv41 import mx8
    v = torch.cat([torch.linspace(-95.0, 25.0, 48000), torch.linspace(-91.5, -85.0, 4000), -torch.logspace(-37.5, 1.9, 5000),
                   torch.logspace(-37.5, 38, 5000), torch.tensor([0.0, -0.0, math.inf, -100.0, -3e38] + [0.0] * 3)])
    v = v[odd:]
    n = v.numel()
    assert (n % 8 != 0) == bool(odd)
    w = mx8.Quantized(torch.zeros(n, 64, dtype=torch.uint8, device=gpu), torch.full((n, 2), 127, dtype=torch.uint8, device=gpu))
    x = mx8.Quantized(torch.zeros(rows, 64, dtype=torch.uint8, device=gpu), torch.full((rows, 2), 127, dtype=torch.uint8, device=gpu))
    got = mx8.MX8Linear(*w, v.to(gpu))(x, activation="silu").double().cpu()
    d = v.double()
    want = d * torch.sigmoid(d)
    fine = want.isfinite()
    assert (got[:, ~fine] == want[~fine]).all()
    size, steps = want[fine].abs(), (32 + 2 * d[fine].abs().clamp(max=1e4)) * 2.0 ** -24
    steps = torch.where(d[fine] > 0, torch.full_like(steps, 64 * 2.0 ** -24), steps)      # 1 + exp(-v): its error counts as exp(-v) does
    near = size * (2.0 ** -8 * (1 + steps) + steps) + 2.0 ** -142 + (size < 2.0 ** -126) * 2.0 ** -126
    off = (got[:, fine] - want[fine]).abs()
    assert (off <= near).all(), (d[fine][(off > near)[0]][:8], (off / size)[off > near][:8])
