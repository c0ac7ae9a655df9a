"""Adapter calls refuse outputs that lie over what other workgroups still read, on the host."""

from __future__ import annotations

import pytest
import torch

BF = torch.bfloat16


@pytest.fixture
def abi(monkeypatch):
    """The wrappers on CPU tensors; the C call returns at once."""
    from dsv41 import _abi
    monkeypatch.setattr(_abi, "_gpu", lambda name, *t: None)
    monkeypatch.setattr(_abi, "_stream", lambda t: None)
    monkeypatch.setattr(_abi, "_call", lambda name, *args: None)
    return _abi


class _Arena:
    """Tensors in turn in one allocation, and views at any byte of it."""

    def __init__(self):
        self.pool, self.end = torch.zeros(1 << 16, dtype=torch.uint8), 0

    def put(self, dtype, *shape):
        self.end = -(-self.end // 16) * 16
        t = self.at(self.end, dtype, *shape)
        self.end += t.numel() * t.element_size()
        return t

    def at(self, first, dtype, *shape):
        n = torch.Size(shape).numel() * torch.empty(0, dtype=dtype).element_size()
        return self.pool[first:first + n].view(dtype).view(shape)

    def place(self, t):
        return t.data_ptr() - self.pool.data_ptr()


def _refused(fn):
    with pytest.raises(ValueError, match="overlaps"):
        fn()


def _operands(arena, n, rank=8, slots=3, k=64, rows=6):
    return dict(x=arena.put(BF, rows, k), w=arena.put(BF, n, k), a=arena.put(BF, slots, rank, k), b=arena.put(BF, slots, n, rank),
                scale=arena.put(torch.float32, slots), ids=arena.put(torch.int32, rows))


def _over(arena, t, rows, n):
    """Outputs [rows, n] that begin with t, end with its first value or begin with its last."""
    size, at = rows * n * 2, arena.place(t)
    end = at + t.numel() * t.element_size()
    return [arena.at(first, BF, rows, n) for first in (at, end - 2, at - size + 2)]


@pytest.mark.parametrize("form", ["adapter_linear", "adapter_plain"])
def test_outputs_over_any_operand(abi, form):
    arena = _Arena()
    arena.end = 4096
    o = _operands(arena, 64)
    call = lambda out: getattr(abi, form)(**o, out=out)                  # noqa: E731
    call(None)
    call(arena.put(BF, 6, 64))
    for name, t in o.items():
        for out in _over(arena, t, 6, 64):
            _refused(lambda: call(out))
    first = arena.at(arena.place(o["x"]) - 6 * 64 * 2, BF, 6, 64)          # right before the first operand
    call(first)


def test_outputs_of_the_pair(abi):
    arena = _Arena()
    arena.end = 4096
    p, q = _operands(arena, 64), _operands(arena, 32)
    x, ids = p["x"], p["ids"]
    bank = lambda o: (o["a"], o["b"], o["scale"])                         # noqa: E731
    out0, out1 = arena.put(BF, 6, 64), arena.put(BF, 6, 32)

    def call(bank0, bank1, out0, out1):
        return abi.adapter_linear_pair(x, p["w"], q["w"], bank0, bank1, ids, out0, out1)

    call(bank(p), bank(q), out0, out1)
    call(bank(p), None, out0, None)
    for t in (x, ids, p["w"], q["w"], *bank(p), *bank(q)):
        for out in _over(arena, t, 6, 64):
            _refused(lambda: call(bank(p), bank(q), out, None))
        for out in _over(arena, t, 6, 32):
            _refused(lambda: call(bank(p), bank(q), None, out))
    _refused(lambda: call(None, bank(q), out0, arena.at(arena.place(out0) + 6 * 64 * 2 - 2, BF, 6, 32)))
    spare = arena.at(arena.place(p["a"]), BF, 6, 64)                        # a bank that the call does not take
    call(None, bank(q), spare, out1)


def test_sums_in_place_or_apart(abi):
    arena = _Arena()
    arena.end = 4096
    o = _operands(arena, 64)
    del o["w"]
    y = arena.put(BF, 6, 64)
    call = lambda out: abi.adapter_add(**o, y=y, out=out)                 # noqa: E731
    assert call(y) is y and call(None).shape == y.shape
    arena.end += 2 * 6 * 64
    call(arena.put(BF, 6, 64))
    at = arena.place(y)
    for shift in (2, 64, 2 * 6 * 64 - 2):
        _refused(lambda: call(arena.at(at + shift, BF, 6, 64)))
        _refused(lambda: call(arena.at(at - shift, BF, 6, 64)))
    call(arena.at(at + 2 * 6 * 64, BF, 6, 64))
    for t in (o["b"], o["scale"], o["ids"]):
        for out in _over(arena, t, 6, 64):
            _refused(lambda: call(out))
    call(o["x"])                                                         # read by the launch before
