"""What the 8-bit projections refuse, on the host: wrong shapes, types, devices, sizes and overlaps reach no kernel."""

from __future__ import annotations

import ctypes

import pytest
import torch

from common import C1, RELEASE_TOY, model_args

BF, U8 = torch.bfloat16, torch.uint8


class _Launched(Exception):
    pass


@pytest.fixture
def host_abi(monkeypatch):
    """The wrappers on CPU tensors, with the C call replaced by a check of its argument count."""
    from dsv41 import _abi

    def fake_call(name, *args):
        assert len(args) == len(_abi._SIGNATURES[name]), name
        raise _Launched(name)

    monkeypatch.setattr(_abi, "_gpu", lambda name, *t: None)
    monkeypatch.setattr(_abi, "_stream", lambda t: None)
    monkeypatch.setattr(_abi, "_call", fake_call)
    return _abi


def _reaches(fn):
    with pytest.raises(_Launched):
        fn()


def _refused(fn, match):
    with pytest.raises(ValueError, match=match):
        fn()


def test_wrappers_refuse_cpu_tensors():
    from dsv41 import mx8
    x = torch.zeros(2, 64, dtype=BF)
    q = mx8.Quantized(torch.zeros(2, 64, dtype=U8), torch.zeros(2, 2, dtype=U8))
    for fn in (lambda: mx8.quantize(x), lambda: mx8.quantize_weight(x), lambda: mx8.dequantize(q),
               lambda: mx8.norm_quantize(x, torch.ones(64), 1e-6), lambda: mx8.MX8Linear(*q)(q)):
        _refused(fn, "GPU")
    with pytest.raises(TypeError):
        mx8.quantize([1.0])


def test_quantization_checks_its_rows(host_abi):
    A = host_abi
    x = torch.zeros(3, 64, dtype=BF)
    _reaches(lambda: A.quant_mx8(x))
    _reaches(lambda: A.quant_mx8(x.float()))
    _reaches(lambda: A.quant_mx8_blocks(x))
    assert A.quant_mx8(x[:0])[1].shape == (0, 2) and A.quant_mx8_blocks(x[:0])[1].shape == (0, 2)
    for f in (A.quant_mx8, A.quant_mx8_blocks):
        _refused(lambda: f(x[:, :48].contiguous()), "whole blocks")
        _refused(lambda: f(x[:, :0]), "whole blocks")
        _refused(lambda: f(torch.zeros((), dtype=BF)), "whole blocks")
        _refused(lambda: f(x[:, :32]), "contiguous")
        _refused(lambda: f(x.half()), "dtype")
        _refused(lambda: f(x, codes=torch.zeros(3, 32, dtype=U8)), "out must be")
        _refused(lambda: f(x, scales=torch.zeros(3, 2, dtype=torch.int8)), "out must be")
    _refused(lambda: A.quant_mx8_blocks(x[None]), "must be")
    both = torch.zeros(3 * 64 + 6, dtype=U8)
    _refused(lambda: A.quant_mx8(x, both[:192].view(3, 64), both[180:186].view(3, 2)), "overlaps")
    _refused(lambda: A.quant_mx8(x, x.view(U8).view(-1)[:192].view(3, 64), both[:6].view(3, 2)), "overlaps")


def test_widths_are_32_bit_numbers(host_abi):
    """A row of 2^32 + 32 channels (memory that is asked for and never touched) is none of 32."""
    k = (1 << 32) + 32
    wide, scales = torch.empty(1, k, dtype=U8), torch.empty(1, k // 32, dtype=U8)
    _refused(lambda: host_abi.dequant_mx8(wide, scales), "fewer than")
    del wide
    x = torch.empty(1, k, dtype=BF)
    _refused(lambda: host_abi.quant_mx8(x), "fewer than")
    _refused(lambda: host_abi.rmsnorm_mx8(x, torch.ones(32), 1e-6), "fewer than")


def test_reading_back_checks_its_codes(host_abi):
    A = host_abi
    c, s = torch.zeros(40, 64, dtype=U8), torch.zeros(40, 2, dtype=U8)
    _reaches(lambda: A.dequant_mx8(c, s))
    _reaches(lambda: A.dequant_mx8(c, s[:2].contiguous(), torch.float32))
    assert A.dequant_mx8(c[:0], s[:0]).shape == (0, 64)
    _refused(lambda: A.dequant_mx8(c, s[:3].contiguous()), "do not go with")
    _refused(lambda: A.dequant_mx8(c, s[:, :1].contiguous()), "do not go with")
    _refused(lambda: A.dequant_mx8(c.view(torch.int8), s), "uint8")
    _refused(lambda: A.dequant_mx8(c[:, :48].contiguous(), s), "whole blocks")
    _refused(lambda: A.dequant_mx8(c[:, :32], s[:, :1].contiguous()), "contiguous")
    _refused(lambda: A.dequant_mx8(c, s, torch.float16), "dtype")
    _refused(lambda: A.dequant_mx8(c, s, out=torch.zeros(40, 32, dtype=BF)), "out must be")
    held = torch.zeros(40 * 64 * 2, dtype=U8)
    _refused(lambda: A.dequant_mx8(held[:2560].view(40, 64), s, out=held.view(BF).view(40, 64)), "overlaps")


def test_norm_checks_its_tensors(host_abi):
    A = host_abi
    x, w = torch.zeros(3, 64, dtype=BF), torch.ones(64)

    def call(**kw):
        args = dict(x=x, weight=w, eps=1e-6)
        args.update(kw)
        return lambda: A.rmsnorm_mx8(**args)

    _reaches(call())
    _reaches(call(delta=x.clone(), rows=False))
    assert A.rmsnorm_mx8(x[:0], w, 1e-6)[0].shape == (0, 64)
    _refused(call(x=x[:, :48].contiguous()), "whole blocks")
    _refused(call(x=x[:, :32], weight=w[:32]), "contiguous")
    _refused(call(weight=w[:32]), "weight")
    _refused(call(weight=w.to(BF)), "weight")
    _refused(call(weight=None), "weight")
    _refused(call(delta=x[:2]), "delta")
    _refused(call(delta=x.float()), "delta")
    _refused(call(delta=torch.zeros(64, 3, dtype=BF).t()), "contiguous")
    _refused(call(delta=x), "overlaps")
    _refused(call(rows=False, out=torch.zeros_like(x)), "not asked for")
    _refused(call(out=x), "overlaps")
    _refused(call(out=torch.zeros(3, 64)), "out must be")
    codes = torch.zeros(3, 64, dtype=U8)
    _refused(call(codes=codes, scales=codes.view(-1)[:6].view(3, 2)), "overlaps")


def test_products_check_their_operands(host_abi):
    A = host_abi
    x, xs = torch.zeros(3, 64, dtype=U8), torch.zeros(3, 2, dtype=U8)
    w, ws = torch.zeros(40, 64, dtype=U8), torch.zeros(2, 2, dtype=U8)

    def call(**kw):
        args = dict(x=x, x_scales=xs, w=w, w_scales=ws)
        args.update(kw)
        return lambda: A.linear_mx8(**args)

    _reaches(call())
    _reaches(call(w_scales=torch.zeros(40, 2, dtype=U8), bias=torch.zeros(40), activation="gelu"))
    y = torch.zeros(3, 40, dtype=BF)
    _reaches(call(residual=y, out=y))
    _reaches(call(x=x.view(1, 3, 64), x_scales=xs.view(1, 3, 2)))
    assert A.linear_mx8(x[:0], xs[:0], w, ws).shape == (0, 40)
    _refused(call(x=x.view(torch.int8)), "uint8")
    _refused(call(x=x[:, :32], x_scales=xs[:, :1].contiguous()), "contiguous")
    _refused(call(x=x[:, :32].contiguous(), x_scales=xs[:, :1].contiguous()), "contract")
    _refused(call(x_scales=xs[:2].contiguous()), "do not go with rows")
    _refused(call(w_scales=ws[:1].contiguous()), "do not go with a weight")
    _refused(call(x=x[0, 0], x_scales=xs[0, 0]), "whole blocks")
    _refused(call(w=w[None]), "must be")
    _refused(call(w=w[:0], w_scales=ws[:0]), "contract")
    many = torch.zeros((1 << 20) + 1, 32, dtype=U8), torch.zeros((1 << 20) + 1, 1, dtype=U8)
    _refused(lambda: A.linear_mx8(*many, torch.zeros(4, 32, dtype=U8), torch.zeros(1, 1, dtype=U8)), "2\\^20")
    _refused(call(bias=torch.zeros(39)), "bias")
    _refused(call(bias=torch.zeros(40, dtype=BF)), "bias")
    _refused(call(activation="tanh"), "activation")
    _refused(call(residual=y.float()), "residual")
    _refused(call(residual=y[:2]), "residual")
    _refused(call(out=y.float()), "out must be")
    held = torch.zeros(7, 40, dtype=BF)
    _refused(call(residual=held[1:4], out=held[2:5]), "overlaps")
    _refused(call(x=held.view(U8).view(-1)[:192].view(3, 64), out=held[:3]), "overlaps")
    w1, ws1 = torch.zeros(8, 64, dtype=U8), torch.zeros(1, 2, dtype=U8)
    _reaches(lambda: A.linear_mx8_pair(x, xs, w, ws, w1, ws1))
    _refused(lambda: A.linear_mx8_pair(x, xs, w, ws, w1, torch.zeros(8, 2, dtype=U8)), "scales over")
    _refused(lambda: A.linear_mx8_pair(x, xs, w, ws, w1[:, :32].contiguous(), ws1), "contract")
    _refused(lambda: A.linear_mx8_pair(x, xs, w, ws, w1, ws1, held[:3], held.view(-1)[100:124].view(3, 8)), "overlaps")


def test_the_library_checks_sizes_before_any_launch():
    from dsv41 import _abi
    lib = _abi.lib()
    at, odd = ctypes.c_void_p(256), ctypes.c_void_p(264)       # never dereferenced: rejected before a launch
    eps = ctypes.c_float(1e-6)

    def message():
        return lib.dsv41_last_error_string()

    for f in (lib.dsv41_quant_mx8, lib.dsv41_quant_mx8_blocks):
        assert f(None, at, at, 1, 32, 1, None) == -1 and b"null" in message()
        assert f(at, at, at, 1, 48, 1, None) == -3
        assert f(at, at, at, 1, 32, 2, None) == -2
        assert f(odd, at, at, 1, 32, 1, None) == -1 and b"aligned" in message()
        assert f(at, at, at, 1 << 30, 32, 1, None) == -3 and b"2^34" in message()
        assert f(at, at, at, -1, 32, 1, None) == -3
        assert f(at, at, at, 0, 32, 1, None) == 0
    assert lib.dsv41_dequant_mx8(at, at, at, 4, 64, 2, 1, None) == -3 and b"1 or 32" in message()
    assert lib.dsv41_dequant_mx8(at, at, at, 0, 64, 32, 1, None) == 0
    assert lib.dsv41_rmsnorm_mx8(at, None, None, None, at, at, 1, 64, eps, 1, None) == -1 and b"weight" in message()
    assert lib.dsv41_rmsnorm_mx8(at, None, at, None, at, at, 1, 16416, eps, 1, None) == -3
    assert lib.dsv41_rmsnorm_mx8(at, None, at, None, at, at, 1 << 24, 32, eps, 1, None) == -3
    assert lib.dsv41_rmsnorm_mx8(at, odd, at, None, at, at, 1, 64, eps, 1, None) == -1 and b"aligned" in message()

    def linear(x=at, w=at, bias=None, residual=None, y=at, rows=1, k=64, n=8, per=32, act=0):
        return lib.dsv41_linear_mx8(x, at, w, at, bias, residual, y, rows, k, n, per, act, None)

    assert linear(rows=0) == 0
    assert linear(x=None) == -1 and b"null" in message()
    assert linear(k=48) == -3 and linear(k=0) == -3 and linear(n=0) == -3 and linear(rows=-1) == -3
    assert linear(k=1 << 21) == -3 and linear(rows=(1 << 20) + 1) == -3 and linear(n=(1 << 24) + 1) == -3
    assert linear(per=2) == -3 and linear(act=4) == -1 and linear(act=-1) == -1
    assert linear(w=odd) == -1 and linear(y=odd) == -1 and linear(residual=odd) == -1 and linear(bias=odd) == -1
    assert linear(rows=1 << 20, n=1 << 24) == -3 and b"too many tiles" in message()
    pair = lib.dsv41_linear_mx8_pair
    assert pair(at, at, at, at, at, at, at, at, 1, 64, 8, 0, 32, None) == -3
    assert pair(at, at, at, at, None, at, at, at, 1, 64, 8, 8, 32, None) == -1
    assert pair(at, at, at, at, at, at, at, at, 0, 64, 8, 8, 32, None) == 0


def test_modules_check_what_they_hold():
    from dsv41 import mx8
    c, s = torch.zeros(40, 64, dtype=U8), torch.zeros(2, 2, dtype=U8)
    lin = mx8.MX8Linear(c, s, torch.zeros(40, dtype=BF))
    assert (lin.in_features, lin.out_features) == (64, 40) and lin.bias.dtype == torch.float32
    assert not any(True for _ in lin.parameters()) and set(lin.state_dict()) == {"codes", "scales", "bias"}
    _refused(lambda: mx8.MX8Linear(c.float(), s), "uint8")
    _refused(lambda: mx8.MX8Linear(c[:, :48], s), "whole blocks")
    _refused(lambda: mx8.MX8Linear(c, s[:1]), "do not go with")
    _refused(lambda: mx8.MX8Linear(c, s, torch.zeros(39)), "bias")
    x = torch.zeros(2, 64, dtype=BF, requires_grad=True)
    for fn in (lambda: mx8.quantize(x), lambda: mx8.quantize_weight(x), lambda: lin(x),
               lambda: mx8.norm_quantize(x, torch.ones(64), 1e-6),
               lambda: mx8.norm_quantize(x.detach(), torch.ones(64), 1e-6, delta=x)):
        _refused(fn, "not differentiable")
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(x.detach(), torch.ones_like(x))
        _refused(lambda: mx8.quantize(dual), "tangent")


def test_layers_check_what_they_hold_in_8_bits():
    from dsv41.attention import Attention
    with pytest.raises(ValueError, match="bfloat16"):
        Attention(0, model_args(C1), torch.float32, "cpu").quantize_projections()
    a = Attention(0, model_args(RELEASE_TOY), BF, "cpu")
    with pytest.raises(ValueError, match="8 bits are for"):
        a.quantize_projections(("wo_a",))
    a.add_adapters(2, 8, ("wq_b",))
    with pytest.raises(ValueError, match="adapters"):
        a.quantize_projections()
    assert not a.takes_quantized
