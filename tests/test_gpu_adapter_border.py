"""Adapter pairs whose first projection ends inside a workgroup's columns: the waves of one workgroup see different
banks, ids that name an adapter in one and none in the other, one adapter or several."""

from __future__ import annotations

import pytest
import torch

from common import SEED_BASE

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


@pytest.mark.parametrize("ids", [[-1] * 9, [4] * 9, [0] * 9, [4, 5, 4, 5, 4, 5, 4, 5, 4], [0, 1, 2, 3, 4, 5, -1, 0, 1]],
                         ids=["none", "second-only", "both-one", "second-several", "mixed"])
@pytest.mark.parametrize("b", [1, 9, 40])
def test_waves_of_both_projections(gpu, ids, b):
    """32 + 64 and 96 + 160 outputs: borders at 32 and 96, in the middle of 64 columns. Values are small integers (x and A
    in {-1, 0, 1}, W and B likewise): every product and sum is exact in float32, the result is rounded once."""
    from dsv41 import _abi
    g = torch.Generator(device="cuda").manual_seed(SEED_BASE + b)
    draw = lambda *s: torch.randint(-1, 2, s, generator=g, device="cuda").to(BF)      # noqa: E731
    ids = torch.tensor((ids * 5)[:b], dtype=torch.int32, device="cuda")
    for n0, n1, slots0, slots1 in ((32, 64, 4, 6), (96, 160, 6, 4)):
        k, r0, r1 = 512, 8, 24
        print(f"[border] b={b} n={n0}+{n1} ids={ids.tolist()}", flush=True)
        x, w0, w1 = draw(b, k), draw(n0, k), draw(n1, k)
        banks = [(draw(s, r, k), draw(s, n, r), torch.arange(1, s + 1, device="cuda").float())
                 for s, n, r in ((slots0, n0, r0), (slots1, n1, r1))]
        for use in ((banks[0], banks[1]), (banks[0], None), (None, banks[1])):
            got = _abi.adapter_linear_pair(x, w0, w1, *use, ids)
            for y, w, bank in zip(got, (w0, w1), use):
                want = x.double() @ w.double().t()
                if bank is not None:
                    a, bb, scale = (t.double() for t in bank)
                    for i, t in enumerate(ids.tolist()):
                        if 0 <= t < len(scale):
                            want[i] += scale[t] * (bb[t] @ (a[t] @ x[i].double()))
                assert torch.equal(y, want.to(BF)), (n0, n1, [u is not None for u in use])
