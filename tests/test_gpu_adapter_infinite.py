"""Infinite values in an adapter's second factor: every form of the call gives what the formula gives, wherever the
rank-wide intermediate is neither zero nor short of bits."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu
BF = torch.bfloat16

# one row, few and many decode rows, split sums of prompts, finished first products, direct tiles; one adapter per tile
# and several; outputs of one 32-column tile and of many
SHAPES = [(1, 1, 512, 64), (6, 1, 512, 64), (30, 1, 512, 256), (20, 1, 1280, 32768), (60, 1, 2048, 640), (100, 1, 512, 96),
          (2, 100, 512, 256), (1, 600, 1024, 512), (50, 6, 256, 512), (3, 333, 1280, 2048), (1, 4144, 1280, 512)]


@pytest.mark.parametrize("rank", [8, 16, 24, 64, 128])
@pytest.mark.parametrize("b,n,k,out", SHAPES)
def test_infinite_second_factor(gpu, b, n, k, out, rank):
    """x A^T is 1 + 2^-12 + 2^-22 for every rank, to the last bit, W is zero: an infinite B gives an infinity of its sign,
    finite ones 0.25 rank times that, opposite infinities NaN; sequences under other adapters stay as they are."""
    from dsv41 import _abi
    print(f"[infinite] b={b} n={n} k={k} out={out} rank={rank}", flush=True)
    x = torch.zeros(b, n, k, dtype=BF, device="cuda")
    x[..., 0], x[..., k // 2], x[..., k - 1] = 1.0, 2.0 ** -12, 2.0 ** -22
    w = torch.zeros(out, k, dtype=BF, device="cuda")
    a = torch.ones(3, rank, k, dtype=BF, device="cuda")
    bb = torch.full((3, out, rank), 0.25, dtype=BF, device="cuda")
    inf = float("inf")
    bb[1, ::4, 0], bb[1, 1::4, rank - 1], bb[1, 2::8, rank // 2] = inf, -inf, inf
    bb[1, 6::8, 0], bb[1, 6::8, 1] = inf, -inf
    ids = torch.arange(b, dtype=torch.int32, device="cuda") % 4 - 1 if b > 1 else torch.ones(1, dtype=torch.int32, device="cuda")
    y = _abi.adapter_linear(x, w, a, bb, torch.ones(3, device="cuda"), ids)
    finite = torch.tensor(0.25 * rank * (1 + 2.0 ** -12 + 2.0 ** -22), device="cuda").to(BF)
    want = torch.zeros(b, out, dtype=BF, device="cuda")
    want[ids >= 0] = finite
    hit = ids == 1
    col = torch.arange(out, device="cuda")
    for pick, value in ((col % 4 == 0, inf), (col % 4 == 1, -inf), (col % 8 == 2, inf), (col % 8 == 6, float("nan"))):
        want[hit[:, None] & pick[None]] = value
    assert torch.equal(y.nan_to_num(nan=7.0, posinf=8.0, neginf=9.0),
                       want[:, None].expand(b, n, out).nan_to_num(nan=7.0, posinf=8.0, neginf=9.0))
