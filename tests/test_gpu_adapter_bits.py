"""The rank-wide intermediate of the adapters counts with all its 24 bits in every form of the call: what is left when
ranks, or the adapter and the projection, cancel. All values and partial sums fit float32, so the result is exact."""

from __future__ import annotations

import pytest
import torch

from test_gpu_adapter_infinite import SHAPES

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


@pytest.mark.parametrize("rank", [8, 16, 24, 64, 128])
@pytest.mark.parametrize("b,n,k,out", SHAPES)
def test_what_cancellation_leaves(gpu, b, n, k, out, rank):
    """x A^T is 1 + 2^-9 + 2^-18 for the first and the last rank, 1 + 2^-9 for the second, x W^T is -3 (1 + 2^-9) for
    every other output: with scale 3, B of 1 and -1 leaves 3 2^-18 of the first two, and of the last and W."""
    from dsv41 import _abi
    print(f"[bits] b={b} n={n} k={k} out={out} rank={rank}", flush=True)
    places = [0, k // 2, k - 1]
    x = torch.zeros(b, n, k, dtype=BF, device="cuda")
    for p, v in zip(places, (1.0, 2.0 ** -9, 2.0 ** -18)):
        x[..., p] = v
    a = torch.zeros(3, rank, k, dtype=BF, device="cuda")
    a[:, 0, places] = a[:, rank - 1, places] = 1.0
    a[:, 1, places[:2]] = 1.0
    bb = torch.zeros(3, out, rank, dtype=BF, device="cuda")
    bb[:, ::2, 0], bb[:, ::2, 1] = 1.0, -1.0
    bb[:, 1::2, rank - 1] = 1.0
    w = torch.zeros(out, k, dtype=BF, device="cuda")
    w[1::2, places[0]] = w[1::2, places[1]] = -3.0
    ids = torch.arange(b, dtype=torch.int32, device="cuda") % 4 - 1 if b > 1 else torch.ones(1, dtype=torch.int32, device="cuda")
    y = _abi.adapter_linear(x, w, a, bb, torch.full((3,), 3.0, device="cuda"), ids)
    want = torch.full((b, out), 3 * 2.0 ** -18, dtype=BF, device="cuda")
    want[ids < 0, ::2], want[ids < 0, 1::2] = 0.0, torch.tensor(-3 * (1 + 2.0 ** -9), device="cuda").to(BF)
    assert torch.equal(y, want[:, None].expand(b, n, out))
