"""Low-rank adapters of many sequences against their formula in 64 bits.

Bounds: products of bf16 values are exact in float32, so a sum of k of them is off by at most k 2^-23 times the sum of
their magnitudes (float32 ones round once more); the rank-wide intermediate carries at least 16 bits into the second
product (2^-16 of its magnitude bound); the result is rounded to its type by at most half a step, twice where the
projection itself is torch's."""

from __future__ import annotations

import pytest
import torch

from common import C1, SEED_BASE, args, load_stack, model_args
from oracle import cpu_ref as R

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32


def _lin(w):
    lin = torch.nn.Linear(1, 1, bias=False)
    lin.weight = torch.nn.Parameter(w, requires_grad=False)
    return lin


def _case(seed, b, n, k, out, rank, slots, dtype=BF, ids=None):
    from dsv41.adapters import AdapterBank
    g = torch.Generator(device="cuda").manual_seed(SEED_BASE + seed)
    normal = lambda *s: torch.randn(*s, generator=g, device="cuda")   # noqa: E731
    lin = _lin((normal(out, k) * k ** -0.5).to(dtype))
    bank = AdapterBank(slots, k, out, rank, dtype)
    for t in range(slots):
        r = max(1, rank - t % 3)                       # adapters of smaller rank among them
        bank.load(t, (normal(r, k) * k ** -0.5).to(dtype), (normal(out, r) * 0.3).to(dtype), 0.5 + 0.25 * t)
    x = normal(b, n, k).to(dtype)
    if ids is None:
        ids = torch.randint(-1, slots, (b,), generator=g, device="cuda")
    return lin, x, bank, torch.as_tensor(ids, device="cuda").to(torch.int32)


def _formula(lin, x, bank, ids):
    """The result in 64 bits and the bound of the float32 work behind it."""
    k, rank = x.shape[-1], bank.a.shape[1]
    xd, w = x.double(), lin.weight.double()
    y, err = xd @ w.t(), k * 2 ** -23 * (xd.abs() @ w.abs().t())
    base = y.clone()
    for i, t in enumerate(ids.tolist()):
        if 0 <= t < bank.slots:
            a, b, s = bank.a[t].double(), bank.b[t].double(), float(bank.scale[t])
            y[i] += s * ((xd[i] @ a.t()) @ b.t())
            most = abs(s) * ((xd[i].abs() @ a.abs().t()) @ b.abs().t())
            err[i] += most * ((k + rank + 4) * 2 ** -23 + 2 ** -16)
    return y, err, base


def _assert_close(got, lin, x, bank, ids):
    y, err, base = _formula(lin, x, bank, ids)
    half = torch.finfo(got.dtype).eps / 2
    err = err + half * (y.abs() + err) + half * (base.abs() + err)
    bad = (got.double() - y).abs() > err
    assert not bad.any(), (int(bad.sum()), float(((got.double() - y).abs() / err).max()))


SHAPES = [
    # decode: one row, odd batches, several 16-row tiles, every projection's kind of shape
    (1, 1, 1280, 512, 16, 4), (3, 1, 512, 96, 8, 2), (17, 1, 640, 1280, 24, 5), (33, 1, 2048, 640, 64, 8),
    (64, 1, 5120, 512, 16, 64), (65, 1, 1280, 2048, 12, 7), (128, 1, 512, 8192, 128, 3), (100, 1, 192, 32, 40, 100),
    # a few tokens per sequence: tiles that hold several sequences
    (5, 3, 512, 256, 16, 3), (2, 64, 320, 96, 8, 2), (25, 5, 256, 128, 16, 6),
    # prompts: one token past the decode rows, odd lengths, several sequences in a tile
    (1, 129, 512, 256, 16, 2), (3, 333, 320, 512, 32, 2), (7, 61, 256, 160, 8, 3), (2, 1000, 1024, 1280, 64, 2),
    (1, 4096, 256, 256, 16, 1), (200, 1, 256, 192, 16, 9), (300, 2, 64, 64, 8, 40),
    # widths and ranks that no tile takes
    (4, 1, 72, 40, 5, 3), (2, 150, 100, 33, 3, 2), (3, 2, 128, 64, 200, 3), (3, 400, 512, 1024, 136, 2),
]


@pytest.mark.parametrize("b,n,k,out,rank,slots", SHAPES)
@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
def test_adapter_linear(gpu, b, n, k, out, rank, slots, dtype):
    from dsv41.adapters import adapter_linear
    print(f"[adapters] b={b} n={n} k={k} out={out} rank={rank} slots={slots} {dtype}", flush=True)
    lin, x, bank, ids = _case(b + n + k, b, n, k, out, rank, slots, dtype)
    got = adapter_linear(lin, x, bank, ids)
    assert got.shape == (b, n, out) and got.dtype == dtype
    _assert_close(got, lin, x, bank, ids)
    assert torch.equal(got, adapter_linear(lin, x, bank, ids))          # the same call again, bit for bit
    flat = adapter_linear(lin, x.view(b * n, k), bank, ids.repeat_interleave(n))
    _assert_close(flat.view(b, n, out), lin, x, bank, ids)


@pytest.mark.parametrize("b,n,k,out", [(9, 1, 512, 256), (33, 1, 1280, 8192), (3, 100, 512, 512), (40, 7, 256, 320)])
def test_rows_without_an_adapter(gpu, b, n, k, out):
    """Slots outside the bank count as none, and what other sequences' adapters hold - NaN, infinities - does not
    reach a row that does not name them."""
    from dsv41.adapters import adapter_linear
    lin, x, bank, _ = _case(b, b, n, k, out, 16, 4)
    none = adapter_linear(lin, x, bank, torch.full((b,), -1, dtype=torch.int32, device="cuda"))
    _assert_close(none, lin, x, bank, torch.full((b,), -1))
    for outside in (4, 1 << 30, -(1 << 31)):
        ids = torch.full((b,), outside, dtype=torch.int32, device="cuda")
        assert torch.equal(adapter_linear(lin, x, bank, ids), none)
    ids = torch.arange(b, device="cuda", dtype=torch.int32) % 5 - 1
    clean = adapter_linear(lin, x, bank, ids)
    bank.a[1].fill_(float("nan"))
    bank.b[2].fill_(float("inf"))
    bank.a[3, :, ::2] = float("-inf")
    got = adapter_linear(lin, x, bank, ids)
    keep = ids <= 0
    assert torch.equal(got[keep], clean[keep]) and torch.equal(got[ids < 0], none[ids < 0])
    assert not got[ids == 1].isfinite().any() and not got[ids == 3].isfinite().any()


def test_infinite_intermediate_gives_the_formula(gpu):
    """x A^T past float32's range: infinity times the finite column of B, in its sign."""
    from dsv41.adapters import adapter_linear
    for n in (1, 150):
        lin, x, bank, ids = _case(3, 2, n, 128, 64, 8, 1, ids=[0, -1])
        x.fill_(1e20)
        bank.a.fill_(0)
        bank.a[0, 0] = 1e19
        bank.b.fill_(0.5)
        bank.b[0, ::2, 0] = -0.5
        bank.b[0, :, 1:] = 1.0
        got = adapter_linear(lin, x, bank, ids)
        want = torch.full((64,), float("inf"), device="cuda")
        want[::2] = float("-inf")
        assert (got[0] == want).all() and got[1].isfinite().all()


@pytest.mark.parametrize("b,n,k,n0,n1,r0,r1", [(1, 1, 1280, 256, 96, 16, 8), (17, 1, 5120, 1280, 512, 8, 8),
                                               (64, 1, 512, 128, 64, 16, 64), (3, 77, 512, 256, 128, 16, 16),
                                               (100, 1, 512, 8192, 512, 16, 24), (1, 1100, 640, 1280, 512, 16, 64),
                                               (7, 300, 1024, 1280, 512, 64, 64), (2, 300, 320, 256, 96, 8, 40),
                                               (2, 2000, 512, 2560, 512, 32, 8),
                                               (2, 2, 72, 40, 24, 4, 4)])
def test_pair_equals_two_projections(gpu, b, n, k, n0, n1, r0, r1):
    from dsv41.adapters import adapter_linear_pair
    lin0, x, bank0, ids = _case(1, b, n, k, n0, r0, 6)
    lin1, _, bank1, _ = _case(2, b, n, k, n1, r1, 3)           # fewer slots: ids 3..5 are none of its own
    got = adapter_linear_pair(lin0, lin1, x, bank0, bank1, ids)
    _assert_close(got[0], lin0, x, bank0, ids)
    _assert_close(got[1], lin1, x, bank1, ids)
    one = adapter_linear_pair(lin0, lin1, x, None, bank1, ids)
    _assert_close(one[0], lin0, x, bank0, torch.full((b,), -1))
    _assert_close(one[1], lin1, x, bank1, ids)
    other = adapter_linear_pair(lin0, lin1, x, bank0, None, ids)
    _assert_close(other[0], lin0, x, bank0, ids)
    _assert_close(other[1], lin1, x, bank1, torch.full((b,), -1))


@pytest.mark.parametrize("b,n", [(5, 1), (2, 140)])
def test_captured_calls_follow_the_ids(gpu, b, n):
    """A captured call reads ids when it is replayed; two graphs hold workspaces of their own; another stream."""
    from dsv41.adapters import adapter_linear
    lin, x, bank, ids = _case(11, b, n, 512, 256, 16, 4)
    eager = lambda: adapter_linear(lin, x, bank, ids)        # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        warm = eager()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(warm, eager())
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = eager()
        graphs.append((g, out))
    for step in range(4):
        ids.copy_((torch.arange(b, device="cuda") + step) % 6 - 1)
        x.mul_(1.25)
        want = eager()
        torch.cuda.synchronize()
        for g, _ in graphs:
            g.replay()
        torch.cuda.synchronize()
        for _, out in graphs:
            assert torch.equal(out, want)
        bank.scale.add_(0.125)


def test_module_call_and_workspace(gpu):
    """Hooks on the projection run; a caller's workspace serves when it is large enough and is refused when it is not
    one; a bank changes between calls."""
    from dsv41 import _abi
    from dsv41.adapters import adapter_linear
    lin, x, bank, ids = _case(5, 4, 1, 512, 256, 16, 4, ids=[0, 1, -1, 3])
    before = adapter_linear(lin, x, bank, ids)
    calls = []
    handle = lin.register_forward_hook(lambda *a: calls.append(1))
    _assert_close(adapter_linear(lin, x, bank, ids), lin, x, bank, ids)
    handle.remove()
    assert calls == [1]
    y = torch.nn.functional.linear(x, lin.weight)
    ws = torch.empty(1 << 16, dtype=torch.uint8, device="cuda")
    assert torch.equal(_abi.adapter_add(x, bank.a, bank.b, bank.scale, ids, y, workspace=ws),
                       _abi.adapter_add(x, bank.a, bank.b, bank.scale, ids, y))
    inplace = y.clone()
    _abi.adapter_add(x, bank.a, bank.b, bank.scale, ids, inplace, out=inplace)
    assert torch.equal(inplace, _abi.adapter_add(x, bank.a, bank.b, bank.scale, ids, y))
    bank.clear(1)
    after = adapter_linear(lin, x, bank, ids)
    assert torch.equal(after[0], before[0]) and not torch.equal(after[1], before[1])
    _assert_close(after, lin, x, bank, ids)
    with pytest.raises(ValueError, match="not differentiable"):
        adapter_linear(lin, x.clone().requires_grad_(), bank, ids)


def test_empty_batch(gpu):
    from dsv41.adapters import adapter_linear
    lin, x, bank, ids = _case(5, 2, 3, 512, 256, 16, 4)
    assert adapter_linear(lin, x[:0], bank, ids[:0]).shape == (0, 3, 256)
    assert adapter_linear(lin, x[:, :0].contiguous(), bank, ids).shape == (2, 0, 256)


def test_stack_with_adapters_equals_merged_weights(gpu, monkeypatch):
    """Two sequences under two adapters through a whole stack - prompt, then single tokens - against one stack each
    whose weights hold w + scale B A; a sequence without adapters against the plain stack. Both sides are within the
    stack's 1e-5 of the exact result."""
    import dsv41.fakequant as FQ
    from dsv41.model import AttentionStack
    monkeypatch.setattr(FQ, "DISABLE", True)
    params = R.make_params(args(C1), SEED_BASE, "f32")

    def stack():
        st = AttentionStack(model_args(C1), F32, gpu)
        load_stack(st, params)
        return st

    g = torch.Generator(device="cuda").manual_seed(SEED_BASE)
    many, merged = stack(), [stack(), stack()]
    for layer, banks in enumerate(many.add_adapters(2, 4)):
        assert set(banks) == {"wq_a", "wkv", "wq_b", "wo_b"}
        for name, bank in banks.items():
            for t in range(2):
                a = torch.randn(4, bank.in_features, generator=g, device="cuda") * bank.in_features ** -0.5
                b = torch.randn(bank.out_features, 4, generator=g, device="cuda") * 0.02
                bank.load(t, a, b, 0.5 + t)
                w = getattr(merged[t].layers[layer], name).weight
                w.copy_((w.double() + (0.5 + t) * (b.double() @ a.double())).float())
    plain = stack()
    with pytest.raises(ValueError, match="without adapters"):
        plain(torch.zeros(1, 1, C1["dim"], device="cuda"), plain.make_cache(1, 64),
              torch.zeros(1, dtype=torch.int32, device="cuda"))
    h = torch.randn(3, 40, C1["dim"], generator=g, device="cuda")
    caches = [st.make_cache(3, 64) for st in (many, *merged, plain)]
    ids = torch.tensor([1, -1, 0], dtype=torch.int32, device="cuda")
    for s, e in ((0, 33), (33, 34), (34, 35), (35, 40)):
        part = h[:, s:e].contiguous()
        got = many(part, caches[0], ids)
        want = [st(part, c) for st, c in zip((*merged, plain), caches[1:])]
        for row, of in ((0, 1), (1, 2), (2, 0)):
            assert (got[row] - want[of][row]).abs().max() <= 2e-5 * max(1.0, float(want[of][row].abs().max()))
        assert (want[0] - want[2]).abs().max() > 1e-3               # the adapters do something


def test_outputs_past_32_bits(gpu):
    """70,000 rows of 32,768 outputs: the last rows of 2.3 billion values, against the formula."""
    from dsv41.adapters import adapter_linear
    lin, x, bank, ids = _case(21, 2, 35000, 64, 32768, 8, 2, ids=[1, 0])
    got = adapter_linear(lin, x, bank, ids)
    assert got.numel() > 1 << 31
    for rows in (slice(0, 3), slice(34990, 35000)):
        _assert_close(got[:, rows].contiguous(), lin, x[:, rows].contiguous(), bank, ids)


def test_add_past_32_bits(gpu):
    """2^20 + 3 rows of 4,096 outputs, more than one launch has threads: the sum taken in turn, in place."""
    from dsv41 import _abi
    rows = (1 << 20) + 3
    g = torch.Generator(device="cuda").manual_seed(23)
    x, a, b = (torch.randint(-3, 4, s, generator=g, device="cuda").to(BF) for s in ((rows, 8), (2, 1, 8), (2, 4096, 1)))
    ids = torch.randint(-1, 2, (rows,), generator=g, device="cuda", dtype=torch.int32)
    y = torch.ones(rows, 4096, dtype=BF, device="cuda")
    assert y.numel() > 1 << 32
    _abi.adapter_add(x, a, b, torch.ones(2, device="cuda"), ids, y, out=y)
    for part in (slice(0, 5), slice(rows - 5, rows)):
        t = ids[part].long()
        h = (x[part].double()[:, None] @ a.double()[t].transpose(1, 2).contiguous())[:, 0]        # small integers
        want = 1 + torch.where(t[:, None] >= 0, h * b.double()[t, :, 0], 0.0)
        assert torch.equal(y[part].double(), want.to(BF).double())


def test_an_output_of_the_callers(gpu):
    from dsv41 import _abi
    lin, x, bank, ids = _case(22, 5, 1, 256, 256, 16, 4)
    want = _abi.adapter_linear(x, lin.weight, bank.a, bank.b, bank.scale, ids)
    out = torch.full((6, 1, 256), 7.0, dtype=BF, device="cuda")
    _abi.adapter_linear(x, lin.weight, bank.a, bank.b, bank.scale, ids, out=out[:5])
    assert torch.equal(out[:5], want) and (out[5] == 7).all()       # the row behind the last sequence
    plain = _abi.adapter_plain(x, lin.weight, bank.a, bank.b, bank.scale, ids, out=out[:5])
    _assert_close(plain, lin, x, bank, ids)
    assert (out[5] == 7).all()
    with pytest.raises(ValueError, match="overlaps"):
        _abi.adapter_linear(x, lin.weight, bank.a, bank.b, bank.scale, ids, out=x)
    with pytest.raises(TypeError):
        _abi.adapter_linear(x, lin.weight, bank.a, bank.b, bank.scale, [0, 1, 2, 3, 0])
