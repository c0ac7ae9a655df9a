"""What the adapter and cache-move entry points refuse, on the host: wrong shapes, types, devices and sizes reach no
kernel. Also the banks' and caches' host logic."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

from common import C1, RELEASE_TOY, model_args

BF = torch.bfloat16


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


def _bank(slots=3, k=64, n=32, rank=8, dtype=BF):
    from dsv41.adapters import AdapterBank
    return AdapterBank(slots, k, n, rank, dtype, "cpu")


def test_loading_leaves_no_graph():
    """Weights that require gradients are copied into a bank, and the bank's tensors follow no graph."""
    b = _bank()
    a0, b0 = torch.randn(4, 64, dtype=BF).requires_grad_(), torch.randn(32, 4, dtype=BF).requires_grad_()
    b.load(1, a0, b0, 0.5)
    assert not (b.a.requires_grad or b.b.requires_grad or b.scale.requires_grad)
    assert torch.equal(b.a[1, :4], a0) and torch.equal(b.b[1, :, :4], b0) and not b.a[1, 4:].any()
    b.clear(1)
    assert not b.a.any() and not b.b.any() and not b.scale.any()


def test_adapter_add_checks_its_tensors(host_abi):
    A, b = host_abi, _bank()
    x, y, ids = torch.zeros(2, 5, 64, dtype=BF), torch.zeros(2, 5, 32, dtype=BF), torch.zeros(2, dtype=torch.int32)

    def call(**kw):
        args = dict(x=x, a=b.a, b=b.b, scale=b.scale, ids=ids, y=y)
        args.update(kw)
        return lambda: A.adapter_add(**args)

    _reaches(call())
    _reaches(call(x=x[:, 0].contiguous(), y=y[:, 0].contiguous()))
    assert A.adapter_add(x[:0], b.a, b.b, b.scale, ids[:0], y[:0]).shape == (0, 5, 32)
    _refused(call(ids=ids.long()), "ids must be int32")
    _refused(call(ids=ids[:1]), "ids must be int32")
    _refused(call(a=b.a[:, :, :32].contiguous()), "no adapters")
    _refused(call(b=b.b[:2]), "no adapters")
    _refused(call(b=b.b[:, :, :4].contiguous()), "no adapters")
    _refused(call(a=b.a.float()), "adapters of")
    _refused(call(scale=b.scale.to(BF)), "scale")
    _refused(call(scale=b.scale[:2]), "scale")
    _refused(call(y=y.float()), "does not go with")
    _refused(call(y=y[:1]), "does not go with")
    _refused(call(x=x.transpose(0, 1)), "contiguous")
    _refused(call(x=x.double()), "adapters of")
    _refused(call(x=x[0, 0]), "x must be")
    _refused(call(out=y.float()), "out must be")
    _refused(call(workspace=torch.zeros(64)), "workspace")
    _refused(call(ids=ids.to("meta")), "tensors on")


def test_adapter_linear_checks_its_tensors(host_abi):
    A, b, c = host_abi, _bank(), _bank(slots=2, n=96, rank=16)
    x, w, ids = torch.zeros(2, 5, 64, dtype=BF), torch.zeros(32, 64, dtype=BF), torch.zeros(2, dtype=torch.int32)
    w1 = torch.zeros(96, 64, dtype=BF)

    def call(**kw):
        args = dict(x=x, w=w, a=b.a, b=b.b, scale=b.scale, ids=ids)
        args.update(kw)
        return lambda: A.adapter_linear(**args)

    _reaches(call())
    _reaches(call(out=torch.zeros(2, 5, 32, dtype=BF), workspace=torch.zeros(1 << 20, dtype=torch.uint8)))
    assert A.adapter_linear(x[:0], w, b.a, b.b, b.scale, ids[:0]).shape == (0, 5, 32)
    with pytest.raises(TypeError):
        A.adapter_linear(x, w, b.a, b.b, b.scale, [0, 1])
    square, c64 = torch.zeros(64, 64, dtype=BF), _bank(n=64)
    _refused(lambda: A.adapter_linear(x, square, c64.a, c64.b, c64.scale, ids, out=x), "overlaps x")
    arena = torch.zeros(40, 64, dtype=BF)                 # input and output side by side in one allocation, or not
    _reaches(lambda: A.adapter_linear(arena[:10], square, c64.a, c64.b, c64.scale, ids.repeat(5), out=arena[10:20]))
    _refused(lambda: A.adapter_linear(arena[:10], square, c64.a, c64.b, c64.scale, ids.repeat(5), out=arena[9:19]),
             "overlaps x")
    _refused(call(x=x[..., :0], a=b.a[..., :0], w=w[:, :0]), "no adapters")
    _refused(call(w=w.float()), "bfloat16")
    _refused(call(w=w1), "no adapters")
    _refused(call(w=torch.zeros(32, 128, dtype=BF)), "contract")
    _refused(call(w=torch.zeros(64, 32, dtype=BF).t()), "contiguous")
    _refused(call(ids=ids[:1]), "ids must be int32")
    _refused(call(out=torch.zeros(2, 5, 32)), "out must be")
    _refused(call(workspace=torch.zeros(64)), "workspace")

    def plain(**kw):
        args = dict(x=x, w=w, a=b.a, b=b.b, scale=b.scale, ids=ids)
        args.update(kw)
        return lambda: A.adapter_plain(**args)

    _reaches(plain())
    assert A.adapter_plain(x[:0], w, b.a, b.b, b.scale, ids[:0]).shape == (0, 5, 32)
    _refused(plain(w=w.float()), "contract")
    _refused(plain(w=w1), "no adapters")
    _refused(plain(out=torch.zeros(2, 5, 32)), "out must be")

    def pair(**kw):
        args = dict(x=x, w0=w, w1=w1, bank0=(b.a, b.b, b.scale), bank1=(c.a, c.b, c.scale), ids=ids)
        args.update(kw)
        return lambda: A.adapter_linear_pair(**args)

    _reaches(pair())
    _reaches(pair(bank0=None))
    _reaches(pair(bank1=None))
    _refused(pair(bank0=None, bank1=None), "no adapters")
    one = torch.zeros(2, 5, 32, dtype=BF)
    _refused(pair(w1=w, bank1=None, out0=one, out1=one), "other output")
    _refused(pair(bank1=(b.a, b.b, b.scale)), "no adapters")
    _refused(pair(w1=w1.float()), "bfloat16")
    _refused(pair(out1=torch.zeros(2, 5, 32, dtype=BF)), "out must be")


def test_cpu_tensors_are_refused():
    from dsv41 import _abi
    b = _bank()
    x, ids = torch.zeros(2, 64, dtype=BF), torch.zeros(2, dtype=torch.int32)
    _refused(lambda: _abi.adapter_add(x, b.a, b.b, b.scale, ids, torch.zeros(2, 32, dtype=BF)), "GPU only")


def test_banks():
    from dsv41.adapters import AdapterBank, adapter_linear
    b = _bank(rank=12)
    assert b.a.shape == (3, 16, 64) and b.b.shape == (3, 32, 16)        # ranks are held in multiples of 8
    b.load(1, torch.ones(12, 64), torch.ones(32, 12), 0.5)
    b.load(1, torch.full((2, 64), 3.0), torch.full((32, 2), 2.0))       # a smaller one leaves nothing of the last
    assert (b.a[1, :2] == 3).all() and not b.a[1, 2:].any() and not b.b[1, :, 2:].any() and b.scale[1] == 1
    assert not b.a[0].any() and not b.a[2].any()
    b.clear(1)
    assert not b.a.any() and not b.b.any() and not b.scale.any()
    for slot in (-1, 3):
        _refused(lambda: b.load(slot, torch.zeros(2, 64), torch.zeros(32, 2)), "slot")
        _refused(lambda: b.clear(slot), "slot")
    _refused(lambda: b.load(0, torch.zeros(13, 64), torch.zeros(32, 13)), "rank at most")
    _refused(lambda: b.load(0, torch.zeros(2, 63), torch.zeros(32, 2)), "no adapter")
    _refused(lambda: b.load(0, torch.zeros(2, 64), torch.zeros(32, 3)), "no adapter")
    for bad in ((0, 64, 32, 8), (1, 0, 32, 8), (1, 64, 0, 8), (1, 64, 32, 0)):
        _refused(lambda: AdapterBank(*bad, device="cpu"), "positive")
    _refused(lambda: AdapterBank(1, 64, 32, 8, torch.float16, "cpu"), "dtype")
    lin = torch.nn.Linear(64, 40, bias=False, dtype=BF)
    lin.register_forward_hook(lambda *a: None)            # the module's own call, which the bank does not go with
    _refused(lambda: adapter_linear(lin, torch.zeros(2, 64, dtype=BF), b, torch.zeros(2, dtype=torch.int32)), "projection")


def test_layers_take_adapters_on_their_projections():
    from dsv41.attention import Attention
    a = Attention(0, model_args(C1), torch.float32, "cpu")
    _refused(lambda: a.add_adapters(2, 4, ("wo_a",)), "wo_a")
    banks = a.add_adapters(2, 4, ("wq_a", "wo_b"))
    assert set(banks) == {"wq_a", "wo_b"} and a.adapters is banks
    assert banks["wo_b"].a.shape == (2, 8, 64) and banks["wo_b"].b.shape == (2, 256, 8)
    assert not any("adapter" in k for k in a.state_dict())


def _cache(bsz=4, cap=40, offset=9, **kw):
    from dsv41.cache import ModelCache
    c = ModelCache(model_args(RELEASE_TOY), bsz, cap, BF, "cpu", **kw)
    c.offset = offset
    return c


def test_moves_check_their_arguments(host_abi):
    from dsv41.cache import copy_sequences, reorder_sequences
    c = _cache()
    _reaches(lambda: reorder_sequences(c, [1, 0, -1]))
    _reaches(lambda: reorder_sequences(c, np.array([1, 0]), torch.tensor([3, 2])))
    _refused(lambda: reorder_sequences(c, [4]), "must lie in")
    _refused(lambda: reorder_sequences(c, [-2]), "must lie in")
    _refused(lambda: reorder_sequences(c, [0], [-1]), "must lie in")
    _refused(lambda: reorder_sequences(c, [0], [4]), "must lie in")
    _refused(lambda: reorder_sequences(c, [0, 1, 2, 3, 0]), "into a cache of 4")
    _refused(lambda: reorder_sequences(c, [0, 1], [2]), "2 moves")
    c.offset = 60
    _refused(lambda: reorder_sequences(c, [1]), "holds")
    c.offset = 9
    other = _cache(bsz=2)
    _reaches(lambda: copy_sequences(other, c, [3], [0]))
    other.offset = 8
    _refused(lambda: copy_sequences(other, c, [3], [0]), "single rows")
    _refused(lambda: copy_sequences(other, c, [3]), "single rows")
    _reaches(lambda: copy_sequences(other, c, [3, 3]))
    assert other.offset == 8                              # a refused or failed move leaves the position
    _refused(lambda: copy_sequences(_cache(cache_format="fp8"), c, [0]), "differ")
    _refused(lambda: copy_sequences(_cache(cache_format="fp8"), _cache(cache_format="fp8", fp8_block_rows=32), [0]), "differ")
    c.layers[1].win_kv = c.layers[1].win_kv[:3]
    _refused(lambda: reorder_sequences(c, [1]), "layer 1")
    c.layers[1].win_kv = c.layers[0].win_kv               # two layers on one buffer, sequences on one row
    _refused(lambda: reorder_sequences(c, [1]), "same memory")
    c.layers[1].win_kv = c.layers[0].win_kv[:1].clone().expand(4, -1, -1)
    _refused(lambda: reorder_sequences(c, [1]), "dense rows")


def test_c_entry_points_refuse_bad_sizes():
    """The library's own checks, without a launch: sizes, types, null pointers, workspaces."""
    from dsv41 import _abi
    lib, p = _abi.lib(), ctypes.c_void_p(4096)

    def add(**kw):
        a = dict(x=p, a=p, b=p, scale=p, ids=p, y=p, out=p, ws=p, bytes=1 << 20, rows=4, tokens=2, k=8, n=8, rank=2,
                 slots=1, dtype=_abi.BF16)
        a.update(kw)
        return lib.dsv41_adapter_add(*a.values(), None)

    assert add(rows=0) == 0
    for bad in (dict(rows=-1), dict(rows=5), dict(tokens=0), dict(k=0), dict(n=0), dict(rank=0), dict(slots=0)):
        assert add(**bad) == -1, bad
    for name in ("x", "a", "b", "scale", "ids", "y", "out"):
        assert add(**{name: None}) == -1, name
    assert add(dtype=_abi.FP8_E4M3) == -2
    assert add(rows=1 << 31, tokens=1) == -1 and add(rows=1 << 30, tokens=1, n=1 << 30) == -1
    assert add(bytes=4 * 2 * 4 - 1) == -4 and add(ws=None) == -4 and add(ws=ctypes.c_void_p(4100)) == -4
    assert lib.dsv41_adapter_add_workspace_bytes(4, 2) == 32
    assert lib.dsv41_adapter_add_workspace_bytes(0, 2) == 0

    def linear(**kw):
        a = dict(x=p, w=p, a=p, b=p, scale=p, ids=p, y=p, ws=p, bytes=1 << 30, rows=4, tokens=2, k=64, n=32, rank=8,
                 slots=1, dtype=_abi.BF16)
        a.update(kw)
        return lib.dsv41_adapter_linear(*a.values(), None)

    assert linear(rows=0) == 0
    for bad in (dict(rows=-1), dict(rows=5), dict(tokens=0), dict(k=0), dict(n=0), dict(rank=0), dict(slots=0),
                dict(slots=-1)):
        assert linear(**bad) == -1, bad
    for name in ("x", "w", "a", "b", "scale", "ids", "y"):
        assert linear(**{name: None}) == -1, name
    for name in ("x", "w", "a", "b", "y"):
        assert linear(**{name: ctypes.c_void_p(4104)}) == -1, name
    assert linear(dtype=_abi.F32) == -2
    for bad in (dict(k=96), dict(n=48), dict(rank=12), dict(rank=136)):
        assert linear(**bad) == -3, bad
    need = lib.dsv41_adapter_linear_workspace_bytes(4, 64, 32, 0, 8, 0)
    assert need > 0 and linear(bytes=need - 1) == -4 and linear(ws=None) == -4
    assert lib.dsv41_adapter_linear_workspace_bytes(0, 64, 32, 0, 8, 0) == 0

    def plain(**kw):
        a = dict(x=p, w=p, a=p, b=p, scale=p, ids=p, y=p, rows=4, tokens=2, k=7, n=5, rank=3, slots=1, dtype=_abi.F32)
        a.update(kw)
        return lib.dsv41_adapter_plain(*a.values(), None)

    assert plain(rows=0) == 0
    for bad in (dict(rows=-1), dict(rows=5), dict(tokens=0), dict(k=0), dict(n=0), dict(rank=0), dict(slots=0),
                dict(rows=1 << 31, tokens=1), dict(rows=1 << 30, tokens=1, n=1 << 20)):
        assert plain(**bad) == -1, bad
    for name in ("x", "w", "a", "b", "scale", "ids", "y"):
        assert plain(**{name: None}) == -1, name
    assert plain(dtype=_abi.FP8_E4M3) == -2

    def pair(**kw):
        a = dict(x=p, w0=p, w1=p, a0=p, b0=p, s0=p, a1=p, b1=p, s1=p, ids=p, y0=p, y1=p, ws=p, bytes=1 << 30, rows=4,
                 tokens=1, k=64, n0=32, n1=32, rank0=8, rank1=8, slots0=1, slots1=1, dtype=_abi.BF16)
        a.update(kw)
        return lib.dsv41_adapter_linear_pair(*a.values(), None)

    assert pair(rows=0) == 0
    assert pair(slots0=0, slots1=0) == -1 and pair(n1=0) == -1 and pair(w1=None) == -1 and pair(y1=None) == -1
    assert pair(a1=None) == -1 and pair(rank1=0) == -1 and pair(rank1=4) == -3
    assert pair(slots0=0, a0=None, b0=None, s0=None, rank0=0, rows=0) == 0

    ptrs = (ctypes.c_void_p * 1)(4096)
    i64 = lambda v: (ctypes.c_int64 * 1)(v)      # noqa: E731
    fill = (ctypes.c_uint32 * 1)(0)

    def move(src=ptrs, dst=ptrs, nbytes=16, buffers=1, order=p, rows=None, moves=1, src_rows=1, dst_rows=1, ws=p,
             size=1 << 20):
        return lib.dsv41_cache_move(src, dst, i64(16), i64(16), i64(nbytes), fill, buffers, order, rows, moves, src_rows,
                                    dst_rows, 1, ws, size, None)

    need = lib.dsv41_cache_move_workspace_bytes(1, 1)
    assert need > 0 and move(size=need - 1) == -4 and move(ws=None) == -4 and move(ws=ctypes.c_void_p(4104)) == -4
    assert lib.dsv41_cache_move_workspace_bytes(0, 1) == lib.dsv41_cache_move_workspace_bytes(1, 0) == 0

    assert move(buffers=0) == 0 and move(moves=0) == 0 and move(nbytes=0) == 0
    for bad in (dict(buffers=-1), dict(moves=-1), dict(src_rows=0), dict(dst_rows=0), dict(nbytes=-1), dict(order=None),
                dict(src=None), dict(dst=None), dict(src=(ctypes.c_void_p * 1)(None)), dict(moves=2)):
        assert move(**bad) == -1, bad
    assert move(moves=4097, rows=p) == -3 and move(dst_rows=4097) == -3
