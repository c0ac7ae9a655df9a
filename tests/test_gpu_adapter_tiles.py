"""Every tile and every second launch of the adapter calls, and the forms off the tiles, on whole numbers: products and
partial sums are exact in float32 in any order, so the result is the formula's, rounded once, to the last bit - or, where
the projection is torch's, its rounded result plus the adapters' part, rounded."""

from __future__ import annotations

import pytest
import torch

from common import SEED_BASE
from test_adapter_plans import CALLS, plan

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32


def _draw(g, top, dtype, *shape):
    return torch.randint(-top, top + 1, shape, generator=g, device="cuda").to(dtype)


def _case(seed, b, n, k, outs, ranks, dtype=BF):
    """x in -3 .. 3, W likewise, A and B in -1 .. 1, scales of 1, 2, -1 and 1/2: a sum of k (at most 8192) products, or of
    rank (128) times 2 k times 3, is a multiple of 1/2 under 2^23."""
    g = torch.Generator(device="cuda").manual_seed(SEED_BASE + seed)
    x, slots = _draw(g, 3, dtype, b, n, k), 5
    w, banks = [], []
    for out, rank in zip(outs, ranks):
        w.append(_draw(g, 3, dtype, out, k))
        scale = torch.tensor([1.0, 2.0, -1.0, 0.5, 2.0], device="cuda")
        banks.append((_draw(g, 1, dtype, slots, rank, k), _draw(g, 1, dtype, slots, out, rank), scale))
    return x, w, banks


def _ids(kind, b):
    ids = {"mixed": torch.arange(b) * 3 % 7 - 1, "one": torch.full((b,), 3), "none": torch.full((b,), -1),
           "half": torch.where(torch.arange(b) < b // 2, 1, -1)}[kind]
    return ids.to(device="cuda", dtype=torch.int32)              # 5 of the mixed ones is no slot


def _part(x, bank, ids):
    a, b, scale = (t.double() for t in bank)
    part = torch.zeros(*x.shape[:2], b.shape[1], dtype=torch.float64, device="cuda")
    for i, t in enumerate(ids.tolist()):
        if 0 <= t < len(scale):
            part[i] = scale[t] * ((x[i].double() @ a[t].t()) @ b[t].t())
    return part


@pytest.mark.parametrize("call", CALLS.values(), ids=lambda c: "-".join(map(str, c)))
@pytest.mark.parametrize("kind", ["mixed", "one", "none", "half"])
def test_every_tile(gpu, call, kind):
    from dsv41 import _abi
    b, n, k, n0, n1, r0, r1 = call
    print(f"[tiles] {call} {plan(*call)} {kind}", flush=True)
    x, w, banks = _case(b + n + k, b, n, k, [n0, n1][:1 + (n1 > 0)], [r0, r1])
    ids = _ids(kind, b)
    if n1:
        got = _abi.adapter_linear_pair(x, *w, *banks, ids)
    else:
        got = (_abi.adapter_linear(x, w[0], *banks[0], ids),)
    for y, wi, bank in zip(got, w, banks):
        want = x.double() @ wi.double().t() + _part(x, bank, ids)
        bad = y.double() != want.to(BF).double()
        assert not bad.any(), (int(bad.sum()), bad.nonzero()[:4].tolist())


@pytest.mark.parametrize("kind", ["mixed", "half"])
@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("b,n,k,out,rank", [(1, 1, 72, 40, 5), (33, 1, 100, 33, 3), (3, 50, 256, 128, 4), (2, 700, 64, 250, 12),
                                            (17, 1, 512, 1280, 136), (6, 40, 96, 1000, 8), (1, 3, 8192, 48, 200)])
def test_the_plain_form_rounds_once(gpu, b, n, k, out, rank, dtype, kind):
    from dsv41 import _abi
    x, (w,), (bank,) = _case(b + n + k, b, n, k, [out], [rank], dtype)
    ids = _ids(kind, b)
    print(f"[plain] {b} {n} {k} {out} {rank} {dtype} {kind}", flush=True)
    want = (x.double() @ w.double().t() + _part(x, bank, ids)).to(dtype)
    assert torch.equal(_abi.adapter_plain(x, w, *bank, ids), want)


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("b,n,k,out,rank", [(1, 1, 64, 32, 8), (7, 5, 100, 33, 3), (2, 300, 512, 640, 136)])
def test_the_sum_on_top_rounds_the_result_only(gpu, b, n, k, out, rank, dtype):
    from dsv41 import _abi
    x, (w,), (bank,) = _case(b + n + k, b, n, k, [out], [rank], dtype)
    ids = _ids("mixed", b)
    y = (x.double() @ w.double().t()).to(dtype)
    print(f"[add] {b} {n} {k} {out} {rank} {dtype}", flush=True)
    assert torch.equal(_abi.adapter_add(x, *bank, ids, y), (y.double() + _part(x, bank, ids)).to(dtype))
