"""Adapter projections have no backward and no forward derivative: every operand that asks for one is refused, whichever
form the call takes. On the host, the kernels replaced by a marker."""

from __future__ import annotations

import pytest
import torch
import torch.autograd.forward_ad as fwAD

BF, F32 = torch.bfloat16, torch.float32


class _Launched(Exception):
    pass


@pytest.fixture(autouse=True)
def abi(monkeypatch):
    from dsv41 import _abi

    def launched(*args, **kw):
        raise _Launched

    for form in ("adapter_linear", "adapter_linear_pair", "adapter_plain", "adapter_add"):
        monkeypatch.setattr(_abi, form, launched)


def _parts(form):
    """x, a projection, a bank and ids whose call takes the named form."""
    from dsv41.adapters import AdapterBank
    dtype = F32 if form == "plain" else BF
    k, n = (64, 32) if form in ("tiles", "add", "bias") else (72, 40)
    lin = torch.nn.Linear(k, n, bias=form == "bias", dtype=dtype).requires_grad_(False)
    if form == "add":
        lin.register_forward_hook(lambda *a: None)
    return torch.randn(2, 3, k).to(dtype), lin, AdapterBank(3, k, n, 8, dtype, "cpu"), torch.zeros(2, dtype=torch.int32)


def _refused(fn):
    with pytest.raises(ValueError, match="not differentiable"):
        fn()


def _reaches(fn):
    with pytest.raises(_Launched):
        fn()


@pytest.mark.parametrize("form", ["tiles", "plain", "add", "bias"])
def test_gradients_wanted(form):
    from dsv41.adapters import adapter_linear
    x, lin, bank, ids = _parts(form)
    call = lambda: adapter_linear(lin, x, bank, ids)             # noqa: E731
    _reaches(call)
    wants = [lin.weight, bank.a, bank.b, bank.scale] + ([lin.bias] if form == "bias" else [])
    for t in wants:
        t.requires_grad_(True)
        _refused(call)
        with torch.no_grad():
            _reaches(call)
        with torch.inference_mode():
            _reaches(call)
        t.requires_grad_(False)
    x.requires_grad_(True)
    _refused(call)


@pytest.mark.parametrize("form", ["tiles", "plain", "add", "bias"])
def test_tangents_held(form):
    from dsv41.adapters import adapter_linear
    x, lin, bank, ids = _parts(form)
    for grad in (torch.enable_grad, torch.no_grad):              # forward derivatives do not ask for gradients
        with grad(), fwAD.dual_level():
            _reaches(lambda: adapter_linear(lin, x, bank, ids))
            _refused(lambda: adapter_linear(lin, fwAD.make_dual(x, torch.ones_like(x)), bank, ids))
            for name in ("a", "b", "scale"):
                plain = getattr(bank, name)
                setattr(bank, name, fwAD.make_dual(plain, torch.ones_like(plain)))
                _refused(lambda: adapter_linear(lin, x, bank, ids))
                setattr(bank, name, plain)
    _reaches(lambda: adapter_linear(lin, x, bank, ids))


def test_the_pair():
    from dsv41.adapters import adapter_linear_pair
    x, lin0, bank0, ids = _parts("tiles")
    _, lin1, bank1, _ = _parts("tiles")
    call = lambda b0, b1: lambda: adapter_linear_pair(lin0, lin1, x, b0, b1, ids)        # noqa: E731
    _reaches(call(bank0, bank1))
    for t in (lin0.weight, lin1.weight, bank0.a, bank0.b, bank0.scale, bank1.a, bank1.b, bank1.scale):
        t.requires_grad_(True)
        _refused(call(bank0, bank1))
        t.requires_grad_(False)
    bank1.b.requires_grad_(True)
    _reaches(call(bank0, None))
    _refused(call(None, bank1))
    bank1.b.requires_grad_(False)
    with fwAD.dual_level():
        bank1.scale = fwAD.make_dual(bank1.scale, torch.ones_like(bank1.scale))
        _refused(call(bank0, bank1))
        _reaches(call(bank0, None))
