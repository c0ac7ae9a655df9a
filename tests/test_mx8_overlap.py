"""The residual addition writes the rows: they may lie over neither the addition nor the norm's weight."""

from __future__ import annotations

import pytest
import torch

from test_mx8_refusals import _reaches, _refused, host_abi          # noqa: F401 (a fixture)


@pytest.mark.parametrize("at", [0, 1, 3])
def test_a_weight_inside_the_rows(host_abi, at):                     # noqa: F811
    x = torch.zeros(4, 64)
    w, d = x.view(-1)[at * 64 + (16 if at < 3 else 0):][:64], torch.zeros(4, 64)
    _refused(lambda: host_abi.rmsnorm_mx8(x, w, 1e-6, d), "overlaps")
    _refused(lambda: host_abi.rmsnorm_mx8(x, w, 1e-6, d, rows=False), "overlaps")
    _reaches(lambda: host_abi.rmsnorm_mx8(x, w, 1e-6))               # only read
    _reaches(lambda: host_abi.rmsnorm_mx8(x, torch.zeros(64), 1e-6, d))
