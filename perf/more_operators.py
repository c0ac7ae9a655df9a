"""Performance cases of the projections in 8 bits, in the form the release stores its weights: e4m3 codes with one
power-of-two scale byte (ue8m0) per 32 x 32 block of a weight and per 32 channels of an activation row.

A case is a dict of plain values; ``op`` says which operator it goes through:

* ``norm``    ``norm_quantize``: a row's residual addition (the row is updated in place), its RMS norm, and the normed row
              in 8 bits, read back;
* ``quant``   ``quantize``: rows in 8 bits, read back (as bf16, which holds every such value);
* ``weight``  ``quantize_weight``: a weight in 32 x 32 blocks, read back;
* ``linear``  ``MX8Linear``: the product of 8-bit rows and an 8-bit weight, with bias, activation and residual;
* ``pair``    ``linear_pair``: two projections of the same rows.

Widths are the released configuration's (hidden 5120, q rank 1280, 64 heads of 512, output rank 8 x 1024), the tiny
float32 configuration's, and others in multiples of 32 channels.
"""

from __future__ import annotations

import math
import os
import sys

import torch

own = False

BF, F32, U8 = torch.bfloat16, torch.float32, torch.uint8
E4M3 = torch.float8_e4m3fn
TYPES = {"bf16": BF, "f32": F32}
EPS = 1e-20
BLOCK, TOP = 32, 448.0                 # channels per scale, the largest e4m3 value
FLOOR = 1e-4                           # the smallest maximum that a block's scale is made for
SHAPES = {"wq_a": (5120, 1280), "wkv": (5120, 512), "wq_b": (1280, 32768), "wo_b": (8192, 5120)}


def _package():
    """The framework's 8-bit projections; its folder is not on the path by itself."""
    root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "deepseek-v41-mlx_amd")
    if root not in sys.path:
        sys.path.insert(0, root)
    from dsv41 import mx8
    return mx8


# ---------------------------------------------------------------------------- the cases


def listed():
    return [
        # one user's token in front of wq_a and wkv: the smallest call, launches and latency
        dict(name="norm_b1", op="norm", rows=1, k=5120, dtype="bf16", delta=True, keep=True),
        # q_norm of an odd decode batch in front of wq_b, nobody else reads the rows
        dict(name="norm_q_b47", op="norm", rows=47, k=1280, dtype="bf16", delta=False, keep=False),
        # a prompt's residual addition and norm
        dict(name="norm_8k", op="norm", rows=8192, k=5120, dtype="bf16", delta=True, keep=True),
        # the output projection's rows of an odd decode batch
        dict(name="quant_b33", op="quant", rows=33, k=8192, dtype="bf16"),
        # float32 rows of an odd number of blocks
        dict(name="quant_f32_1000x4064", op="quant", rows=1000, k=4064, dtype="f32"),
        # the widest projection's weight as it is loaded
        dict(name="weight_wq_b", op="weight", rows=32768, k=1280, dtype="bf16"),
        # one user's token through wq_a and wkv
        dict(name="pair_b1", op="pair", rows=1, k=5120, n=1280, n2=512, bias=False, act="none", residual=False),
        # a full decode batch on the widest projection
        dict(name="wq_b_b64", op="linear", rows=64, k=1280, n=32768, bias=False, act="none", residual=False),
        # an odd decode batch on the output projection, added to the residual stream
        dict(name="wo_b_b33", op="linear", rows=33, k=8192, n=5120, bias=False, act="none", residual=True),
        # three short prompts of an odd length
        dict(name="wq_b_3x333", op="linear", rows=999, k=1280, n=32768, bias=False, act="none", residual=False),
        # a width that no tile divides, with everything the epilogue has
        dict(name="odd_777", op="linear", rows=777, k=2336, n=1111, bias=True, act="silu", residual=True),
        # two long prompts on the output projection: the largest call
        dict(name="wo_b_8k", op="linear", rows=8192, k=8192, n=5120, bias=False, act="none", residual=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("norm", "quant", "weight", "linear", "linear", "linear", "pair"))
    if op in ("norm", "quant", "weight"):
        while True:
            c = dict(op=op, rows=_log(rng, 1, 16384), k=rng.choice((5120, 1280, 512, 8192, BLOCK * _log(rng, 1, 256))),
                     dtype=rng.choice(("bf16", "bf16", "f32")))
            if op == "norm":
                c.update(delta=rng.random() < 0.6, keep=rng.random() < 0.6)
            if c["rows"] * c["k"] <= 8192 * 5120:
                return c
    while True:
        rows = _log(rng, 1, 128) if rng.random() < 0.5 else _log(rng, 129, 8192)
        k, n = rng.choice((SHAPES["wq_a"], SHAPES["wkv"], SHAPES["wq_b"], SHAPES["wo_b"],
                           (BLOCK * _log(rng, 1, 256), _log(rng, 16, 16384))))
        c = dict(op=op, rows=rows, k=k, n=n)
        if op == "pair":
            c["n2"] = rng.choice((512, _log(rng, 16, 4096)))
        c.update(bias=rng.random() < 0.3, act=rng.choice(("none", "none", "none", "relu", "silu", "gelu")),
                 residual=rng.random() < 0.5)
        if op == "pair":
            c.update(bias=False, act="none", residual=False)
        if k * (n + c.get("n2", 0)) <= 1 << 26 and rows * k * (n + c.get("n2", 0)) <= 8192 * 8192 * 5120:
            return c


# ---------------------------------------------------------------------------- the plain form


def _scaled(v):
    """Blocks (the last dimension) of float32 values as e4m3 values and the power of two that goes with each: the
    smallest for which the block's largest value is at most 448."""
    m, e = torch.frexp(v.abs().amax(-1, keepdim=True).clamp(min=FLOOR) * (1.0 / TOP))
    e = e - (m == 0.5).to(e.dtype)
    return (v * torch.exp2(-e.float())).to(E4M3), e


def _rows_8(x):
    """Codes and scale bytes of rows."""
    c, e = _scaled(x.float().view(*x.shape[:-1], x.shape[-1] // BLOCK, BLOCK))
    return c.view(x.shape).view(U8), (e[..., 0] + 127).to(U8)


def _weight_8(w):
    """Codes and scale bytes of a weight in 32 x 32 blocks, the last block of rows perhaps a part of one."""
    n, k = w.shape
    v = torch.nn.functional.pad(w.float(), (0, 0, 0, -n % BLOCK))
    v = v.view(-1, BLOCK, k // BLOCK, BLOCK).transpose(1, 2).reshape(-1, k // BLOCK, BLOCK * BLOCK)
    c, e = _scaled(v)
    c = c.view(U8).view(-1, k // BLOCK, BLOCK, BLOCK).transpose(1, 2).reshape(-1, k)
    return c[:n].contiguous(), (e[..., 0] + 127).to(U8)


def _values(codes, scales):
    """What codes and scale bytes stand for, in 32 bits (exact)."""
    s = torch.exp2(scales.float() - 127.0).repeat_interleave(BLOCK, -1)
    if scales.shape[:-1] != codes.shape[:-1]:
        s = s.repeat_interleave(BLOCK, 0)[:codes.shape[0]]
    return codes.view(E4M3).float() * s


def _activated(y, act):
    if act == "relu":
        return y.clamp(min=0.0)
    if act == "silu":
        return y / (1.0 + torch.exp(-y))
    if act == "gelu":
        return 0.5 * y * (1.0 + torch.erf(y * math.sqrt(0.5)))
    return y


def _product(x, w, bias, act, residual):
    y = torch.matmul(x, w.t())
    if bias is not None:
        y = y + bias
    y = _activated(y, act)
    if residual is not None:
        y = y + residual.float()
    return y.to(BF)


def _normed(h, delta, weight, keep):
    """The row with its addition (in place), normed, and the normed row in 8 bits: each of the rows' type, as the next
    reader takes it."""
    if delta is not None:
        h.copy_(h.float() + delta.float())
    v = h.float()
    y = (weight * (v * (1.0 / torch.sqrt(v.square().mean(-1, keepdim=True) + EPS)))).to(h.dtype)
    values = _values(*_rows_8(y)).to(BF)
    return dict(h=h, values=values, **(dict(y=y) if keep else {}))


# ---------------------------------------------------------------------------- the interface


def _inputs(c, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, scale=1.0):
        return torch.randn(*shape, generator=g, device="cuda").mul_(scale)

    def rows(k):
        """Rows whose channels differ in size, a few of them by far."""
        x = normal(c["rows"], k)
        return x.mul_(torch.exp(normal(k, scale=0.5))).mul_(1.0 + 15.0 * (torch.rand(k, generator=g, device="cuda") < 0.01))

    k = c["k"]
    if c["op"] == "weight":
        return dict(w=normal(c["rows"], k, scale=0.02).to(TYPES[c["dtype"]]))
    if c["op"] in ("norm", "quant"):
        t = TYPES[c["dtype"]]
        s = dict(x=rows(k).to(t))
        if c["op"] == "norm":
            s["delta"] = normal(c["rows"], k, scale=0.3).to(t) if c["delta"] else None
            s["norm"] = 1.0 + normal(k, scale=0.1)
        return s
    s = dict(x=_rows_8(rows(k).to(BF)), w=[_weight_8(normal(n, k, scale=0.02).to(BF))
                                          for n in ((c["n"], c["n2"]) if c["op"] == "pair" else (c["n"],))])
    s["bias"] = normal(c["n"], scale=0.5) if c["bias"] else None
    s["residual"] = normal(c["rows"], c["n"]).to(BF) if c["residual"] else None
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if own and "w" in s and case["op"] != "weight":
        mx8 = _package()
        s["x"] = mx8.Quantized(*s["x"])
        s["lin"] = [mx8.MX8Linear(codes, scales, s["bias"]) for codes, scales in s["w"]]
    s["case"] = case
    return s


def run(state):
    s, c = state, state["case"]
    op = c["op"]
    if own:
        mx8 = _package()
        if op == "norm":
            y, q = mx8.norm_quantize(s["x"], s["norm"], EPS, delta=s["delta"], rows=c["keep"])
            return dict(h=s["x"], values=mx8.dequantize(q), **(dict(y=y) if c["keep"] else {}))
        if op == "quant":
            return mx8.dequantize(mx8.quantize(s["x"]))
        if op == "weight":
            return mx8.dequantize(mx8.quantize_weight(s["w"]))
        if op == "pair":
            return mx8.linear_pair(s["lin"][0], s["lin"][1], s["x"])
        return s["lin"][0](s["x"], activation=c["act"], residual=s["residual"])
    if op == "norm":
        return _normed(s["x"], s["delta"], s["norm"], c["keep"])
    if op == "quant":
        return _values(*_rows_8(s["x"])).to(BF)
    if op == "weight":
        return _values(*_weight_8(s["w"])).to(BF)
    x = _values(*s["x"])
    y = tuple(_product(x, _values(*w), s["bias"], c["act"], s["residual"]) for w in s["w"])
    return y if op == "pair" else y[0]


def work(case):
    c = case
    rows, k = c["rows"], c["k"]
    if c["op"] in ("norm", "quant", "weight"):
        size, parts = TYPES[c["dtype"]].itemsize, 1                         # the rows in
        if c["op"] == "norm":
            parts += (2 if c["delta"] else 0) + (1 if c["keep"] else 0)     # the addition in, the sum out; the normed rows
        return {"bytes": (size * parts + 2) * rows * k + (4 * k if c["op"] == "norm" else 0), "flops": 0}   # values: bf16
    n = c["n"] + c.get("n2", 0)
    moved = rows * (k + k // BLOCK) + n * k + -(-n // BLOCK) * (k // BLOCK) + 2 * rows * n
    moved += (2 * rows * n if c["residual"] else 0) + (4 * n if c["bias"] else 0)
    return {"bytes": moved, "flops": 2 * rows * k * n}


# ---------------------------------------------------------------------------- in 64 bits


def _to_e4m3(v):
    """The nearest e4m3 value (ties to even): steps of an eighth of the value's power of two, of 2^-9 below 2^-6."""
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6))) - 3.0)
    return torch.round(v / step) * step


def _quantized(v, whole):
    """Values in 8 bits, block by block: 32 channels of a row, or 32 x 32 of a weight."""
    out = v.clone()
    high = BLOCK if whole else 1
    n, k = v.shape
    size = v.abs().view(n, k // BLOCK, BLOCK).amax(-1)
    if whole:
        size = torch.stack([part.amax(0) for part in size.split(high)])
    need = size.clamp(min=FLOOR) / TOP
    power = torch.round(torch.log2(need))
    power = torch.where(torch.exp2(power) >= need, power, power + 1.0)      # the smallest power of two at or over `need`
    power = torch.where(torch.exp2(power - 1.0) >= need, power - 1.0, power)
    scale = torch.exp2(power).repeat_interleave(BLOCK, 1).repeat_interleave(high, 0)[:n]
    return _to_e4m3(out / scale) * scale


def _decoded(codes, scales):
    """e4m3 codes from their bits: sign, four bits of exponent (bias 7), three of mantissa."""
    c = codes.long()
    e, m = (c >> 3) & 15, (c & 7).double()
    v = torch.where(e > 0, (1.0 + m / 8.0) * torch.exp2(e.double() - 7.0), m / 8.0 * 2.0 ** -6)
    v = torch.where(c >= 128, -v, v)
    row = torch.arange(codes.shape[0], device=codes.device)
    s = torch.exp2(scales.double() - 127.0)[row if scales.shape[0] == codes.shape[0] else row // BLOCK]
    return (v.view(codes.shape[0], -1, BLOCK) * s[..., None]).view(codes.shape)


def exact(case, seed):
    c, s = case, _inputs(case, seed)
    if c["op"] == "quant":
        return _quantized(s["x"].double(), False)
    if c["op"] == "weight":
        return _quantized(s["w"].double(), True)
    if c["op"] == "norm":
        t = s["x"].dtype
        h = s["x"].double() if s["delta"] is None else s["x"].double() + s["delta"].double()
        v = h.to(t).double()                                                # the residual stream is of the rows' type
        y = s["norm"].double() * v / (v.square().mean(-1, keepdim=True) + EPS).sqrt()
        found = dict(h=h, values=_quantized(y.to(t).double(), False))       # and so is the row that is quantized
        return dict(found, y=y) if c["keep"] else found
    found, x = [], _decoded(*s["x"])
    for w in s["w"]:
        y = x @ _decoded(*w).t()
        if s["bias"] is not None:
            y = y + s["bias"].double()
        if c["act"] == "relu":
            y = torch.where(y > 0, y, torch.zeros_like(y))
        elif c["act"] == "silu":
            y = y * torch.sigmoid(y)
        elif c["act"] == "gelu":
            y = y * 0.5 * torch.special.erfc(-y * math.sqrt(0.5))
        found.append(y if s["residual"] is None else y + s["residual"].double())
    return tuple(found) if c["op"] == "pair" else found[0]
