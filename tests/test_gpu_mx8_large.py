"""Rows and products in 8 bits at the sizes' far end: tensors past 2^32 values, pairs over large tiles, streams side by side and
graphs of large tiles."""

from __future__ import annotations

import pytest
import torch

from test_gpu_mx8 import check, operands, product, spread

pytestmark = pytest.mark.gpu

BF = torch.bfloat16


def same(a, b):
    return all(torch.equal(u, v) for u, v in zip(a, b))


def test_rows_past_32_bits(gpu):
    """Codes, scales, read-back values and normed rows whose place is past 2^32 values: the last rows come out as they do alone,
    and so do the rows about every multiple of 2^31 values."""
    from dsv41 import mx8
    k = 8224
    rows = (1 << 32) // k + 301
    x = torch.empty(rows, k, dtype=BF, device=gpu)
    for at in range(0, rows, 1 << 16):
        x[at:at + (1 << 16)].normal_()
    spots = [0, (1 << 31) // k - 1, (1 << 32) // k - 1, rows - 3]
    q = mx8.quantize(x)
    for r in spots:
        assert same(mx8.quantize(x[r:r + 3]), (q.codes[r:r + 3], q.scales[r:r + 3])), r
    back = mx8.dequantize(q)
    for r in spots:
        assert torch.equal(mx8.dequantize(mx8.Quantized(q.codes[r:r + 3], q.scales[r:r + 3])), back[r:r + 3]), r
    del back
    weight = torch.rand(k, device=gpu) + 0.5
    want = [mx8.norm_quantize(x[r:r + 3].clone(), weight, 1e-6, x[r:r + 3].clone()) for r in spots]
    y, n = mx8.norm_quantize(x, weight, 1e-6, x.clone())
    for r, (v, u) in zip(spots, want):
        assert torch.equal(y[r:r + 3], v) and same((n.codes[r:r + 3], n.scales[r:r + 3]), u), r


def test_weights_past_32_bits(gpu):
    """Blocks of a weight past 2^32 values and their products."""
    from dsv41 import mx8
    k = 8224
    n = ((1 << 32) // k // 32 + 9) * 32 + 5
    w = torch.empty(n, k, dtype=BF, device=gpu)
    for at in range(0, n, 1 << 16):
        w[at:at + (1 << 16)].normal_()
    q = mx8.quantize_weight(w)
    parts = [(0, 64), ((1 << 31) // k // 32 * 32, 64), ((1 << 32) // k // 32 * 32, 64), (n - 37, 37)]     # whole blocks
    for r, m in parts:
        assert same(mx8.quantize_weight(w[r:r + m]), (q.codes[r:r + m], q.scales[r // 32:r // 32 + 2])), r
    del w
    x = mx8.quantize(spread((3, k), 60).to(gpu))
    y, back = mx8.MX8Linear(*q)(x), mx8.dequantize(q)
    for r, m in parts:
        part = mx8.Quantized(q.codes[r:r + m], q.scales[r // 32:r // 32 + 2])
        check(y[:, r:r + m], *product(x, part))
        assert torch.equal(mx8.dequantize(part), back[r:r + m]), r


@pytest.mark.parametrize("k,n", [(8224, 64), (64, 16400), (128, 16401), (512, 16640)])
def test_products_past_32_bits(gpu, k, n):
    """Rows past 2^32 codes, and results past 2^32 values, of few outputs and of whole tiles, with the residual in place."""
    from dsv41 import mx8
    rows = (1 << 32) // max(k, n) + 301
    x, w = operands(300, k, n, 61)
    big = mx8.Quantized(torch.zeros(rows, k, dtype=torch.uint8, device=gpu), torch.full((rows, k // 32), 127, dtype=torch.uint8, device=gpu))
    spots = [0, (1 << 31) // max(k, n) - 150, rows - 300]
    for r in spots:
        big.codes[r:r + 300], big.scales[r:r + 300] = x
    lin = mx8.MX8Linear(*w)
    y, size = product(x, w)
    got = lin(big)
    for r in spots:
        check(got[r:r + 300], y, size)
    res = got[spots[-1]:].clone()
    lin(big, residual=got, out=got)
    check(got[spots[-1]:], y, size, residual=res)


@pytest.mark.parametrize("rows,k,n0,n1,kernel", [(600, 288, 3008, 1111, 1), (2048, 544, 264, 8000, 1), (700, 1056, 5001, 330, 1),
                                                 (400, 512, 1280, 520, 2), (400, 512, 1281, 521, 2), (400, 544, 1281, 521, 2),
                                                 (259, 608, 9000, 4625, 2), (1300, 1024, 7017, 6600, 3),
                                                 (1300, 1024, 6017, 6700, 3), (2100, 640, 5000, 2571, 3)])
def test_a_pair_over_tiles(gpu, rows, k, n0, n1, kernel):
    from dsv41 import _abi, mx8
    assert _abi.linear_mx8_plan(rows, k, n0, n1).kernel == kernel
    x, w0 = operands(rows, k, n0, 62)
    _, w1 = operands(1, k, n1, 63)
    lin0, lin1 = mx8.MX8Linear(*w0), mx8.MX8Linear(*w1)
    held = [torch.full((rows * n + 512,), 7.0, dtype=BF, device=gpu) for n in (n0, n1)]
    y0, y1 = (h[:rows * n].view(rows, n) for h, n in zip(held, (n0, n1)))
    _abi.linear_mx8_pair(*x, lin0.codes, lin0.scales, lin1.codes, lin1.scales, y0, y1)
    check(y0, *product(x, w0))
    check(y1, *product(x, w1))
    assert all((h[rows * n:] == 7.0).all() for h, n in zip(held, (n0, n1)))


@pytest.mark.parametrize("rows,k,n", [(1410, 640, 11001), (1281, 1024, 14001), (130, 640, 5449), (2353, 384, 5019)])
def test_nothing_beyond_large_outputs_is_written(gpu, rows, k, n):
    from dsv41 import _abi
    x, w = operands(rows, k, n, 64)
    held = torch.full((rows * n + 4096,), 7.0, dtype=BF, device=gpu)
    out = held[:rows * n].view(rows, n)
    _abi.linear_mx8(*x, *w, out=out)
    assert (held[rows * n:] == 7.0).all()
    check(out, *product(x, w))


def test_streams_side_by_side(gpu):
    """Calls on two streams at once share nothing: each gives what it gives alone."""
    from dsv41 import mx8
    sizes = [(1410, 640, 11001), (40, 1280, 4096), (1281, 640, 1552)]
    calls = []
    for i, (rows, k, n) in enumerate(sizes):
        x, w = operands(rows, k, n, 65 + i)
        calls.append((mx8.MX8Linear(*w), x, mx8.dequantize(x)))
    want = [(lin(x), mx8.quantize(h)) for lin, x, h in calls]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in calls]
    got = [[] for _ in calls]
    for _ in range(5):
        for s, (lin, x, h), out in zip(streams, calls, got):
            with torch.cuda.stream(s):
                out.append((lin(x), mx8.quantize(h)))
    torch.cuda.synchronize()
    for outs, (y, q) in zip(got, want):
        for y1, q1 in outs:
            assert torch.equal(y1, y) and same(q1, q)


def test_graphs_of_large_tiles(gpu):
    """Two graphs of the same layers over the same buffers, replayed in turn with eager calls between: every replay gives the eager
    results of the rows that it finds."""
    from dsv41 import mx8
    rows = 1410
    lins = [mx8.MX8Linear(*operands(1, k, n, 70 + i)[1]) for i, (k, n) in enumerate([(640, 11008), (640, 1552)])]
    back = mx8.MX8Linear(*operands(1, 11008, 640, 72)[1])
    h, w = spread((rows, 640), 73).to(gpu), torch.rand(640, device=gpu) + 0.5

    def run():
        y, x = mx8.norm_quantize(h, w, 1e-6)
        a, b = mx8.linear_pair(*lins, x)
        return y, a, b, back(a, "silu", residual=h)

    side = torch.cuda.Stream()
    graphs, outs = [], []
    torch.cuda.synchronize()
    for _ in range(2):
        with torch.cuda.stream(side):
            run()
            side.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                outs.append(run())
        graphs.append(graph)
    for turn in range(4):
        h.copy_(spread((rows, 640), 80 + turn).to(gpu))
        want = run()
        torch.cuda.synchronize()
        graphs[turn % 2].replay()
        torch.cuda.synchronize()
        for a, b in zip(outs[turn % 2], want):
            assert torch.equal(a, b)


def test_hooks_run_in_a_pair(gpu):
    """A pair with hooks on one of them calls both, so that the hook sees its product."""
    from dsv41 import mx8
    x, w0 = operands(5, 64, 40, 90)
    _, w1 = operands(1, 64, 33, 91)
    lin0, lin1 = mx8.MX8Linear(*w0), mx8.MX8Linear(*w1)
    want = mx8.linear_pair(lin0, lin1, x)
    seen = []
    handle = lin1.register_forward_hook(lambda m, i, y: seen.append(y))
    got = mx8.linear_pair(lin0, lin1, x)
    handle.remove()
    assert len(seen) == 1 and torch.equal(seen[0], want[1]) and same(got, want)
