"""Rows and weights in 8 bits, the norm that ends in them and their products, against plain implementations in 64 bits.

Codes, scales and read-back values are exact. The products' bound: half a bf16 step of the result (2^-8 of it), and what the
block-scaled instruction cuts off. It sums eight neighbouring channels at a time: products are lined up at the largest of
the eight, and of each what lies under 2^-13 of that one's power of two is cut off (one product at 2^0 and another at 2^-13
in its eight give both, at 2^-14 the first alone; in other eights products count down to float32's last bit). So each of the
seven others loses less than 2^-13 of the largest, which is at most the eight's sum |x w|: 7 * 2^-13 of it in all."""

from __future__ import annotations

import math

import pytest
import torch

from mx8_sizes import SIZES

pytestmark = pytest.mark.gpu

BF, F32 = torch.bfloat16, torch.float32
E4M3 = torch.float8_e4m3fn
HALF = {BF: 2.0 ** -8, F32: 2.0 ** -24}      # half a step, relative
SUMS = 7 * 2.0 ** -13                        # the instruction's sums, of sum |x w|


# ---------------------------------------------------------------------------- the plain forms


def encode(v):
    """Codes and scale bytes [..., blocks] of finite float64 blocks [..., blocks, values]."""
    amax = v.abs().amax(-1).clamp(min=float(torch.tensor(1e-4, dtype=F32)))
    e = torch.ceil(torch.log2(amax / 448.0)).clamp(min=-140.0)
    e = torch.where(torch.exp2(e - 1) * 448.0 >= amax, e - 1, e)
    e = torch.where(torch.exp2(e) * 448.0 < amax, e + 1, e)
    return (v / torch.exp2(e)[..., None]).float().to(E4M3).view(torch.uint8), (e + 127).to(torch.uint8)


def rows_8(x):
    c, s = encode(x.double().cpu().view(*x.shape[:-1], x.shape[-1] // 32, 32))
    return c.view(x.shape), s


def blocks_8(w):
    n, k = w.shape
    v = torch.zeros(-(-n // 32) * 32, k, dtype=torch.float64)
    v[:n] = w.double().cpu()
    c, s = encode(v.view(-1, 32, k // 32, 32).transpose(1, 2).reshape(-1, k // 32, 1024))
    return c.view(-1, k // 32, 32, 32).transpose(1, 2).reshape(-1, k)[:n], s


def decode(codes, scales):
    s = torch.exp2(scales.double().cpu() - 127.0).repeat_interleave(32, -1)
    if scales.shape[:-1] != codes.shape[:-1]:
        s = s.repeat_interleave(32, 0)[:codes.shape[0]]
    return codes.cpu().view(E4M3).double() * s


def spread(shape, seed, dtype=BF, powers=6):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(*shape, generator=g) * torch.exp2(torch.randint(-powers, powers + 1, shape, generator=g).float())
    return x.to(dtype)


def activated(y, act):
    if act == "relu":
        return y.clamp(min=0)
    if act == "silu":
        return y * torch.sigmoid(y)
    if act == "gelu":
        return 0.5 * y * torch.special.erfc(-y * math.sqrt(0.5))
    return y


# ---------------------------------------------------------------------------- quantization


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("shape", [(1, 32), (3, 96), (2, 5, 64), (33, 8192), (100, 4064), (7, 1, 1280), (0, 64)])
def test_rows_are_the_formulas_codes(gpu, shape, dtype):
    from dsv41 import _abi, mx8
    x = spread(shape, 1, dtype).to(gpu)
    q = mx8.quantize(x)
    codes, scales = rows_8(x)
    assert torch.equal(q.scales.cpu(), scales) and torch.equal(q.codes.cpu(), codes)
    for t in (BF, F32):
        assert torch.equal(mx8.dequantize(q, t).cpu().double(), decode(codes, scales))
    if x.numel():                            # the round trip that the fake quantization does
        assert torch.equal(mx8.dequantize(q, dtype), _abi.fq_fp8_ue8m0(x, 32))


@pytest.mark.parametrize("dtype", [BF, F32])
def test_rows_at_the_borders(gpu, dtype):
    """Zero blocks, magnitudes under the floor, maxima at and beside 448 times a power of two, ties, both ends of the type."""
    from dsv41 import mx8
    x = torch.zeros(12, 64, dtype=F32)
    x[1] = 1e-30
    x[2, :32] = torch.linspace(-1, 1, 32)
    x[2, 5] = 448.0
    x[3, 0], x[3, 32] = 448.0 * 2 ** 20, -448.0 * 2 ** -20
    x[4, 0], x[4, 40] = 450.0, 446.0
    x[5, :32] = torch.arange(32) * 0.5 + 16.25           # ties of the e4m3 grid at the scale 2^-3
    x[5, 0] = 56.0
    x[6, 0], x[6, 1] = 3.3e38, -3.3e38
    x[7, 0], x[7, 1] = 1.2e-38, -1e-40
    x[8, :32] = 2.0 ** -9 * torch.arange(32)             # the subnormal grid and its ties
    x[8, 0] = 448.0
    x[9, :32] = 2.0 ** -10 * torch.arange(32)
    x[9, 0] = 448.0
    x[10] = -0.0
    x[11, 63] = -1e-4
    x = x.to(dtype).to(gpu)
    q = mx8.quantize(x)
    codes, scales = rows_8(x)
    assert torch.equal(q.scales.cpu(), scales) and torch.equal(q.codes.cpu(), codes)
    if dtype == F32:
        up = torch.nextafter(torch.tensor(448.0), torch.tensor(1e9))
        down = torch.nextafter(torch.tensor(448.0), torch.tensor(0.0))
        y = torch.stack([up, torch.tensor(448.0), down])[:, None] * 2.0 ** torch.arange(-20, 100, 3.0)
        y = torch.nn.functional.pad(y.reshape(-1, 1), (0, 31)).to(gpu)
        assert torch.equal(mx8.quantize(y).scales.cpu(), rows_8(y)[1])


@pytest.mark.parametrize("dtype", [BF, F32])
def test_blocks_that_are_not_finite(gpu, dtype):
    from dsv41 import mx8
    x = spread((4, 128), 2, dtype)
    x[0, 5], x[1, 33], x[2, 127] = math.nan, math.inf, -math.inf
    bad = torch.zeros(4, 4, dtype=torch.bool)
    bad[0, 0] = bad[1, 1] = bad[2, 3] = True
    q = mx8.quantize(x.to(gpu))
    got = mx8.dequantize(q, F32).cpu()
    wide = bad.repeat_interleave(32, 1)
    assert torch.equal(q.scales.cpu() == 255, bad) and torch.equal(got.isnan(), wide)
    fine = torch.where(wide, torch.zeros(()), x.float())
    codes, scales = rows_8(fine)
    assert torch.equal(got[~wide].double(), decode(codes, scales)[~wide])
    w = spread((40, 64), 3, dtype)
    w[35, 40] = math.inf
    q = mx8.quantize_weight(w.to(gpu))
    assert q.scales.cpu().tolist()[1][1] == 255 and int((q.scales == 255).sum()) == 1
    assert mx8.dequantize(q).cpu().isnan().nonzero().tolist() == [[r, c] for r in range(32, 40) for c in range(32, 64)]


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("n,k", [(1, 32), (31, 64), (32, 256), (33, 288), (100, 1280), (512, 5120), (70, 8192)])
def test_weights_are_the_formulas_blocks(gpu, n, k, dtype):
    from dsv41 import mx8
    w = spread((n, k), 4, dtype, 3).to(gpu)
    q = mx8.quantize_weight(w)
    codes, scales = blocks_8(w)
    assert torch.equal(q.scales.cpu(), scales) and torch.equal(q.codes.cpu(), codes)
    assert torch.equal(mx8.dequantize(q).cpu().double(), decode(codes, scales))


def test_every_code_reads_back(gpu):
    from dsv41 import mx8
    codes = torch.arange(256, dtype=torch.uint8).view(8, 32).repeat(1, 5)
    scales = torch.tensor([0, 1, 100, 127, 255], dtype=torch.uint8).repeat(8, 1)
    want = decode(codes, scales)
    want[:, -32:] = math.nan
    q = mx8.Quantized(codes.to(gpu), scales.to(gpu))
    assert torch.equal(mx8.dequantize(q, F32).cpu().double().nan_to_num(7e7), want.float().double().nan_to_num(7e7))
    assert torch.equal(mx8.dequantize(q).cpu().nan_to_num(7e7), want.to(BF).nan_to_num(7e7))


# ---------------------------------------------------------------------------- norm


def normed(x, w, eps, d=None):
    """The residual addition, rounded (through float32) to the rows' type, and its norm in 64 bits."""
    h = x if d is None else (x.double() + d.double()).to(x.dtype)
    v = h.double()
    return h, w.double() * v / (v.square().mean(-1, keepdim=True) + eps).sqrt()


def nearest(y, want):
    """bf16 rows are the formula's values rounded through float32. float32 rows are within 1/2 + 2^-20 of a step: the root's low
    part is rounded at 2^-48 of it, each product's error at 2^-24 of at most 2^-23 of the product, three such sums for each of
    two products, so under 2^-44 in all, 2^-20 of a step or less; 2^-19 leaves room for the 64 bits' own roundings."""
    if y.dtype is BF:
        return torch.equal(y, want.to(BF))
    half = torch.exp2(torch.floor(torch.log2(want.abs().clamp(min=2.0 ** -126))) - 24)
    return bool(((y.double() - want).abs() <= half * (1 + 2.0 ** -19)).all())


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("rows,dim", [(1, 32), (3, 64), (257, 1280), (5, 5120), (2, 8192), (3, 9248), (2, 16384), (0, 64)])
@pytest.mark.parametrize("add", [False, True])
def test_norm_is_the_two_steps(gpu, rows, dim, dtype, add):
    from dsv41 import mx8
    x, d = spread((rows, dim), 5, dtype, 3), spread((rows, dim), 6, dtype, 3)
    w = 1.0 + 0.2 * torch.randn(dim, generator=torch.Generator().manual_seed(7))
    h = (x.double() + d.double()).to(dtype) if add else x
    v = h.double()
    want = w.double() * v / (v.square().mean(-1, keepdim=True) + 1e-20).sqrt()
    xg, dg = x.to(gpu), d.to(gpu) if add else None
    y, q = mx8.norm_quantize(xg, w.to(gpu), 1e-20, dg)
    if add and dtype == F32:
        h = (x + d)
    assert torch.equal(xg.cpu(), h)
    assert nearest(y.cpu(), want)
    codes, scales = mx8.quantize(y)
    assert torch.equal(q.codes, codes) and torch.equal(q.scales, scales)
    none, q2 = mx8.norm_quantize(x.to(gpu), w.to(gpu), 1e-20, dg, rows=False)
    assert none is None and torch.equal(q2.codes, codes) and torch.equal(q2.scales, scales)


def test_norm_and_the_separate_norms(gpu):
    """The separate norms sum in float32: their rows are at most a step of bf16 off."""
    from dsv41 import _abi, mx8
    x, d = spread((65, 5120), 8).to(gpu), spread((65, 5120), 9).to(gpu)
    w = torch.rand(5120, device=gpu)
    h = x.clone()
    y = _abi.add_rmsnorm(h, d, w, 1e-6)
    got, _ = mx8.norm_quantize(x, w, 1e-6, d)
    assert torch.equal(x, h) and ((got.float() - y.float()).abs() <= y.float().abs() * 2 * HALF[BF]).all()


@pytest.mark.parametrize("rows", [1023, 1024, 2051])
@pytest.mark.parametrize("dim", [32, 512, 544, 1024, 1280, 1536, 2048, 2080])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_norm_of_many_narrow_rows(gpu, rows, dim, dtype):
    """A wave per row and four waves per row: both the formula's rows."""
    from dsv41 import mx8
    x, d = spread((rows, dim), 11, dtype).to(gpu), spread((rows, dim), 12, dtype).to(gpu)
    w = torch.rand(dim, device=gpu) + 0.5
    eps = 2.0 ** -20                             # the same number in 32 bits
    _, want = normed(x, w, eps)
    y, q = mx8.norm_quantize(x, w, eps)
    assert nearest(y, want) and all(torch.equal(a, b) for a, b in zip(q, mx8.quantize(y)))
    h, want = normed(x, w, eps, d)
    y, q = mx8.norm_quantize(x, w, eps, d)
    assert torch.equal(x, h) and nearest(y, want) and all(torch.equal(a, b) for a, b in zip(q, mx8.quantize(y)))


@pytest.mark.parametrize("dtype", [BF, F32])
def test_norm_of_very_large_and_very_small_rows(gpu, dtype):
    """Squares past float32's range on both sides, a row of zeros, and weights that are zero."""
    from dsv41 import mx8
    x = spread((6, 320), 13, dtype, 1).to(gpu)
    x[0] *= 1e30
    x[1] *= 1e-30
    x[2] = 0.0
    w = torch.rand(320, device=gpu) + 0.5
    w[3:5] = 0.0
    for eps in (0.0, 2.0 ** -20):
        y, q = mx8.norm_quantize(x.clone(), w, eps)
        want = normed(x, w, eps)[1]
        if eps == 0.0:
            assert y[2].isnan().all() and want[2].isnan().all()          # 0 / 0
            y[2] = want[2] = 0.0
        assert nearest(y, want)
        assert torch.equal(y.signbit(), want.signbit()) and torch.equal(q.codes[3:], mx8.quantize(y).codes[3:])


def test_norm_of_a_row_that_is_not_finite(gpu):
    from dsv41 import mx8
    x = spread((3, 128), 10).to(gpu)
    want, q0 = mx8.norm_quantize(x.clone(), torch.ones(128, device=gpu), 1e-6)
    x[1, 7] = math.nan
    y, q = mx8.norm_quantize(x, torch.ones(128, device=gpu), 1e-6)
    assert y[1].isnan().all() and (q.scales[1] == 255).all() and mx8.dequantize(q)[1].isnan().all()
    for i in (0, 2):
        assert torch.equal(y[i], want[i]) and torch.equal(q.codes[i], q0.codes[i])


# ---------------------------------------------------------------------------- products


def operands(rows, k, n, seed, per=32):
    from dsv41 import mx8
    x = mx8.quantize(spread((rows, k), seed, BF, 4).cuda())
    w = (spread((n, k), seed + 1, BF, 2) * 0.05).cuda()
    return x, mx8.quantize_weight(w) if per == 32 else mx8.quantize(w)


def product(x, w):
    """The product in 64 bits and sum |x w|."""
    a, b = decode(*x).cuda(), decode(*w).cuda()
    return a @ b.t(), a.abs() @ b.abs().t()


def check(got, y, size, bias=None, act=None, residual=None):
    if bias is not None:
        y, size = y + bias.double(), size + bias.double().abs()
    want = activated(y, act)
    if residual is not None:
        want = want + residual.double()
    # silu and gelu change by at most 1.13 times their argument's change; expf and erff by a few float32 steps of the value
    near = want.abs() * HALF[BF] + 1.13 * SUMS * size * (1 + HALF[BF]) + 2.0 ** -20 * activated(y, act).abs() + 1e-37
    assert got.dtype is BF and got.shape == want.shape
    assert ((got.double() - want).abs() <= near).all(), float(((got.double() - want).abs() / near).max())


@pytest.mark.parametrize("rows", [1, 15, 16, 17, 33, 64, 65, 130, 300])
@pytest.mark.parametrize("k,n", [(32, 32), (64, 1), (96, 5), (128, 100), (160, 33), (1280, 1000), (2336, 1111), (5120, 48)])
def test_products(gpu, rows, k, n):
    from dsv41 import mx8
    x, w = operands(rows, k, n, 20)
    check(mx8.MX8Linear(*w)(x), *product(x, w))


@pytest.mark.parametrize("rows,k,n", [(1, 5120, 1792), (64, 1280, 32768), (33, 8192, 5120), (333, 1280, 8192),
                                      (1000, 512, 5120), (2048, 1280, 2048), (4100, 416, 3000)])
def test_products_of_the_released_widths(gpu, rows, k, n):
    from dsv41 import mx8
    x, w = operands(rows, k, n, 22)
    check(mx8.MX8Linear(*w)(x), *product(x, w))


@pytest.mark.parametrize("rows,k,n", [(1, 64, 40), (37, 288, 65), (130, 1280, 520), (700, 640, 1030), (1100, 256, 2560)])
@pytest.mark.parametrize("act", [None, "relu", "silu", "gelu"])
@pytest.mark.parametrize("per,bias,residual", [(32, True, True), (32, False, True), (1, True, False), (1, False, False)])
def test_epilogues(gpu, rows, k, n, act, per, bias, residual):
    from dsv41 import mx8
    x, w = operands(rows, k, n, 24, per)
    b = torch.randn(n, device=gpu) if bias else None
    r = spread((rows, n), 26).to(gpu) if residual else None
    lin = mx8.MX8Linear(*w, b)
    got = lin(x, activation=act, residual=r)
    check(got, *product(x, w), b, act, r)
    if residual:                             # the residual stream in place
        assert lin(x, activation=act, residual=r, out=r) is r and torch.equal(r, got)


@pytest.mark.parametrize("act", ["relu", "silu", "gelu"])
@pytest.mark.parametrize("rows", [1, 70])
def test_activations_alone(gpu, act, rows):
    """Products of zeros, so that the bias is what is activated: values of every size, both signs, in aligned rows and not."""
    from dsv41 import mx8
    g = torch.Generator().manual_seed(25)
    v = torch.cat([torch.randn(4000, generator=g) * torch.exp2(torch.randint(-20, 5, (4000,), generator=g).float()),
                   torch.linspace(-120, 120, 4801), torch.tensor([0.0, -0.0, 1e30, -1e30, 3e38, -3e38, 1e-30, -1e-30])])
    for n in (v.numel(), v.numel() - v.numel() % 8):
        w = mx8.Quantized(torch.zeros(n, 64, dtype=torch.uint8, device=gpu), torch.full((n, 2), 127, dtype=torch.uint8, device=gpu))
        x = mx8.Quantized(torch.zeros(rows, 64, dtype=torch.uint8, device=gpu), torch.full((rows, 2), 127, dtype=torch.uint8, device=gpu))
        got = mx8.MX8Linear(*w, v[-n:].to(gpu))(x, activation=act).double().cpu()
        d = v[-n:].double()
        want = {"relu": d.clamp(min=0), "silu": d * torch.sigmoid(d), "gelu": 0.5 * d * torch.special.erfc(-d * math.sqrt(0.5))}[act]
        # bf16's half step; gelu's formula is 1.5e-7 off in erf, so 0.75e-7 |v|, and as much again for float32's roundings; silu's
        # exponential is |v| + 2 steps of 2^-24 off and its reciprocal 0 from exp(87) on, where v / exp(87) is under 2e-36
        near = want.abs() * HALF[BF] + {"relu": 0.0, "silu": 2e-36, "gelu": 1.5e-7}[act] * d.abs().clamp(max=1e3 if act == "gelu" else 1.0)
        if act == "silu":
            near = near + want.abs() * (d.abs() + 4.0) * 2.0 ** -24
        assert ((got - want).abs() <= near).all(), (d[(got - want).abs() > near][:8], got[0][((got - want).abs() > near)[0]][:8])


@pytest.mark.parametrize("rows,k,n", SIZES)
def test_every_tile_shape(gpu, rows, k, n):
    """Each shape's products, its last tiles where nothing divides, and its epilogue with the residual stream in place; the
    same bits on every call."""
    from dsv41 import mx8
    x, w = operands(rows, k, n, 28)
    y, size = product(x, w)
    lin = mx8.MX8Linear(*w, torch.randn(n, device=gpu))
    r = spread((rows, n), 29).to(gpu)
    want = lin(x, activation="silu", residual=r)
    check(want, y, size, lin.bias, "silu", r)
    assert lin(x, activation="silu", residual=r, out=r) is r and torch.equal(r, want)
    got = mx8.MX8Linear(*w)(x)
    check(got, y, size)
    assert torch.equal(got, mx8.MX8Linear(*w)(x))


@pytest.mark.parametrize("per", [1, 32])
@pytest.mark.parametrize("rows,k,n", [(444, 640, 4912), (300, 544, 1701), (130, 672, 5449), (141, 608, 10917), (259, 1056, 13625),
                                      (79, 3392, 905), (1324, 1024, 11017)])
def test_scales_off_words(gpu, rows, k, n, per):
    """Scales that begin anywhere in memory, in tensors that end with their last byte."""
    from dsv41 import _abi
    x, w = operands(rows, k, n, 27, per)
    want = product(x, w)
    for off in (1, 2, 3):
        held = [torch.full((t.numel() + off * (i + 1),), 255, dtype=torch.uint8, device=gpu) for i, t in enumerate((x.scales, w.scales))]
        for i, (h, t) in enumerate(zip(held, (x.scales, w.scales))):
            h[off * (i + 1):] = t.flatten()
        xs, ws = (h[off * (i + 1):].view(t.shape) for i, (h, t) in enumerate(zip(held, (x.scales, w.scales))))
        check(_abi.linear_mx8(x.codes, xs, w.codes, ws), *want)


@pytest.mark.parametrize("rows", [1, 16, 40, 200, 1024])
@pytest.mark.parametrize("k,n0,n1", [(64, 1, 1), (256, 96, 33), (5120, 1280, 512)])
def test_a_pair_is_its_two_products(gpu, rows, k, n0, n1):
    from dsv41 import mx8
    x, w0 = operands(rows, k, n0, 30)
    _, w1 = operands(1, k, n1, 31)
    lin0, lin1 = mx8.MX8Linear(*w0), mx8.MX8Linear(*w1)
    y0, y1 = mx8.linear_pair(lin0, lin1, x)
    check(y0, *product(x, w0))
    check(y1, *product(x, w1))
    again = mx8.linear_pair(lin0, lin1, x)
    assert torch.equal(again[0], y0) and torch.equal(again[1], y1)


@pytest.mark.parametrize("rows", [1, 40, 700])
def test_nothing_beyond_the_outputs_is_written(gpu, rows):
    from dsv41 import _abi
    x, w = operands(rows, 160, 77, 33)
    held = torch.full((rows * 77 + 256,), 7.0, dtype=BF, device=gpu)
    out = held[:rows * 77].view(rows, 77)
    _abi.linear_mx8(*x, *w, out=out)
    assert (held[rows * 77:] == 7.0).all()
    check(out, *product(x, w))


@pytest.mark.parametrize("rows", [3, 70, 600])
def test_what_is_not_a_number_stays_where_it_is(gpu, rows):
    """A NaN scale or code of a row reaches that row's outputs alone, of a weight its own columns."""
    from dsv41 import mx8
    x, w = operands(rows, 160, 80, 34)
    want = mx8.MX8Linear(*w)(x)
    x.scales[1, 2] = 255
    w.codes[70, 159] = 0x7F
    got = mx8.MX8Linear(*w)(x)
    bad = torch.zeros(rows, 80, dtype=torch.bool, device=gpu)
    bad[1], bad[:, 70] = True, True
    assert torch.equal(got.isnan(), bad) and torch.equal(got[~bad], want[~bad])


def test_extreme_scales(gpu):
    """2^-127 to 2^127: products that neither overflow nor vanish, ones that do, and results that cancel."""
    from dsv41 import mx8
    codes = torch.full((4, 128), 0x38, dtype=torch.uint8, device=gpu)              # ones
    low, high = torch.zeros(4, 4, dtype=torch.uint8, device=gpu), torch.full((4, 4), 254, dtype=torch.uint8, device=gpu)
    assert (mx8.MX8Linear(codes, high)(mx8.Quantized(codes, low)) == 128.0).all()
    assert (mx8.MX8Linear(codes, high)(mx8.Quantized(codes, high)) == math.inf).all()
    assert (mx8.MX8Linear(codes, low)(mx8.Quantized(codes, low)) == 0.0).all()
    signs = codes.clone()
    signs[:, 64:] = 0xB8
    assert (mx8.MX8Linear(signs, high)(mx8.Quantized(codes, low)) == 0.0).all()


# ---------------------------------------------------------------------------- together


def test_a_layers_projections_together(gpu):
    """A block's residual addition and norm, two projections of it, the norm of one and its projection, and a projection
    back onto the residual stream: each step against its own formula in 64 bits, eager and replayed from a graph."""
    from dsv41 import mx8
    g = torch.Generator(device=gpu).manual_seed(40)
    rows, dim, rank, wide = 9, 320, 96, 256

    def normal(*shape, scale=1.0):
        return (torch.randn(*shape, generator=g, device=gpu) * scale).to(BF)

    def lin(n, k):
        return mx8.MX8Linear(*mx8.quantize_weight(normal(n, k, scale=0.05)))

    qa, kv, qb, back = lin(rank, dim), lin(64, dim), lin(wide, rank), lin(dim, wide)
    w0, w1 = torch.rand(dim, generator=g, device=gpu) + 0.5, torch.rand(rank, generator=g, device=gpu) + 0.5
    h, delta = normal(rows, dim), normal(rows, dim)

    def layer():
        _, x = mx8.norm_quantize(h, w0, 1e-6, delta, rows=False)
        a, b = mx8.linear_pair(qa, kv, x)
        _, r = mx8.norm_quantize(a, w1, 1e-6, rows=False)
        c = qb(r)
        q = mx8.quantize(c)
        return x, a, b, r, q, back(q, residual=h)

    h0 = h.clone()
    x, a, b, r, q, out = layer()
    assert torch.equal(h, (h0.float() + delta.float()).to(BF))
    check(a, *product(x, (qa.codes, qa.scales)))
    check(b, *product(x, (kv.codes, kv.scales)))
    check(out, *product(q, (back.codes, back.scales)), residual=h)

    for t in (h0, delta):
        assert t.isfinite().all()
    side = torch.cuda.Stream()
    h.copy_(h0)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        graph = torch.cuda.CUDAGraph()
        layer()
        side.synchronize()
        with torch.cuda.graph(graph, stream=side):
            got = layer()
    for seed in range(3):
        h0 = (h0 * 0.5 + seed).to(BF)
        h.copy_(h0)
        want = layer()
        want = [torch.cat([t.flatten().view(torch.uint8) for t in (v if isinstance(v, tuple) else (v,))]).clone() for v in want]
        h.copy_(h0)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for v, u in zip(got, want):
            assert torch.equal(torch.cat([t.flatten().view(torch.uint8) for t in (v if isinstance(v, tuple) else (v,))]), u)


def test_float_rows_are_quantized_on_the_way_in(gpu):
    from dsv41 import mx8
    x = spread((5, 3, 160), 41).to(gpu)
    lin = torch.nn.Linear(160, 40, dtype=BF, device=gpu)
    m = mx8.MX8Linear.from_linear(lin)
    assert torch.equal(m(x), m(mx8.quantize(x))) and m(x).shape == (5, 3, 40)
    assert torch.equal(m.weight_values(), mx8.dequantize(mx8.quantize_weight(lin.weight.detach())))
    check(m(x).view(15, 40), *product([t.reshape(15, -1) for t in mx8.quantize(x)], (m.codes, m.scales)), m.bias)
    m2 = mx8.MX8Linear(m.codes, m.scales)
    pair = mx8.linear_pair(m, m2, x)
    assert torch.equal(pair[0], m(x)) and torch.equal(pair[1], m2(x))


def test_no_rows(gpu):
    from dsv41 import mx8
    _, w = operands(1, 64, 40, 42)
    lin = mx8.MX8Linear(*w)
    assert lin(torch.zeros(0, 64, dtype=BF, device=gpu)).shape == (0, 40)
    assert mx8.linear_pair(lin, lin, torch.zeros(2, 0, 64, dtype=BF, device=gpu))[1].shape == (2, 0, 40)


def test_a_call_on_another_stream(gpu):
    """The kernels run on the caller's stream: inputs produced there just before are the ones multiplied."""
    from dsv41 import mx8
    x, w = operands(40, 1280, 4096, 43)
    lin = mx8.MX8Linear(*w)
    want = lin(x)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        codes, scales = torch.zeros_like(x.codes), torch.zeros_like(x.scales)
        big = torch.randn(4096, 4096, device=gpu) @ torch.randn(4096, 4096, device=gpu)
        codes.copy_(x.codes + (big[0, 0] * 0).to(torch.uint8))
        scales.copy_(x.scales)
        got = lin(mx8.Quantized(codes, scales))
    side.synchronize()
    assert torch.equal(got, want)
