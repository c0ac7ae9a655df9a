"""Which projections the adapter calls stand in for, on the host: every module that torch's Linear may be is taken, by
a kernel where its call is the product alone, else by the module's own call and the adapters' part on top."""

from __future__ import annotations

import pytest
import torch

F32 = torch.float32


@pytest.fixture
def forms(monkeypatch):
    """The names of the forms that ran; the sums on top come from the formula."""
    from dsv41 import _abi
    seen = []

    def add(x, a, b, scale, ids, y, out=None, workspace=None):
        seen.append("add")
        return y

    def plain(x, w, a, b, scale, ids, out=None):
        seen.append("plain")
        return x @ w.t()

    monkeypatch.setattr(_abi, "adapter_add", add)
    monkeypatch.setattr(_abi, "adapter_plain", plain)
    return seen


def _linear(bias=False):
    return torch.nn.Linear(24, 40, bias=bias, dtype=F32).requires_grad_(False)


class _Doubled(torch.nn.Linear):
    def forward(self, x):
        return 2 * super().forward(x)


def _tensors(lin, names):
    for name in names:
        t = getattr(lin, name).detach()
        delattr(lin, name)
        setattr(lin, name, t)
    return lin


def _own_forward(lin):
    lin.forward = lambda x: torch.nn.functional.linear(x, lin.weight) + 1
    return lin


@pytest.mark.parametrize("make,form", [
    (lambda: _linear(), "plain"),
    (lambda: _linear(bias=True), "add"),
    (lambda: _tensors(_linear(), ["weight"]), "add"),
    (lambda: _tensors(_linear(bias=True), ["weight", "bias"]), "add"),
    (lambda: _tensors(_linear(bias=True), ["bias"]), "add"),
    (lambda: _Doubled(24, 40, bias=False).requires_grad_(False), "add"),
    (lambda: _own_forward(_linear()), "add"),
    (lambda: torch.nn.utils.parametrizations.orthogonal(_linear()).requires_grad_(False), "add"),
], ids=["linear", "bias", "weight-a-tensor", "both-tensors", "bias-a-tensor", "subclass", "own-forward", "parametrized"])
def test_every_linear(forms, make, form):
    from dsv41.adapters import AdapterBank, adapter_linear, adapter_linear_pair
    lin, x = make(), torch.randn(2, 3, 24)
    bank, ids = AdapterBank(2, 24, 40, 8, F32, "cpu"), torch.zeros(2, dtype=torch.int32)
    want = lin(x)
    assert torch.equal(adapter_linear(lin, x, bank, ids), want) and forms == [form]
    got = adapter_linear_pair(lin, _linear(), x, bank, bank, ids)
    assert torch.equal(got[0], want) and forms == [form, form, "plain"]
