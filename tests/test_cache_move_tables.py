"""The table of a cache's buffers that moves of sequences keep: whatever happens to the cache between two calls, the next
one moves what a table built on the spot lists. On the host."""

from __future__ import annotations

import copy
import pickle
import types

import pytest
import torch

from common import RELEASE_TOY, model_args

BF = torch.bfloat16


@pytest.fixture
def moved(monkeypatch):
    """Moves on CPU caches; gives what reached the C call: its tables as lists."""
    from dsv41 import _abi, cache

    def call(src, dst, src_strides, dst_strides, nbytes, fills, order, rows, src_rows, dst_rows, same, device):
        seen.append([list(t) for t in (src, dst, src_strides, dst_strides, nbytes, fills)] + [src_rows, dst_rows])

    seen = []
    monkeypatch.setattr(_abi, "cache_move", call)

    def move(c):
        cache.reorder_sequences(c, [1, 0])
        return seen.pop()

    return move


def _cache(bsz=4, cap=40, offset=9, **kw):
    from dsv41.cache import ModelCache
    c = ModelCache(model_args(RELEASE_TOY), bsz, cap, BF, "cpu", **kw)
    c.offset = offset
    return c


def _fresh(move, c):
    kept = c.__dict__.pop("_row_table", None)
    want = move(c)
    if kept is not None:
        c._row_table = kept
    return want


def test_whatever_is_assigned(moved):
    from dsv41.compressor import CompressorState
    c = _cache()
    first = moved(c)
    assert first == _fresh(moved, c) and moved(c) == first
    bare, owner = c.layers[0], next(lc for lc in c.layers if lc.comp_state is not None)

    def buffer():
        return torch.zeros(4, 40, 64, dtype=BF)

    steps = [
        ("a buffer for a layer that had none", lambda: setattr(c.layers[3], "comp_kv", buffer())),
        ("another format's buffer", lambda: setattr(c.layers[3], "index_k", buffer())),
        ("a state for a layer that had none", lambda: setattr(c.layers[4], "comp_state", CompressorState(4, 2, 64, "cpu"))),
        ("a state's tensor", lambda: setattr(c.layers[4].comp_state, "kv_state", torch.ones(4, 2, 64))),
        ("a state exchanged", lambda: setattr(owner, "comp_state", CompressorState(4, owner.ratio, 64, "cpu"))),
        ("a state taken away", lambda: setattr(owner, "comp_state", None)),
        ("a buffer exchanged", lambda: setattr(bare, "win_kv", bare.win_kv.clone())),
        ("a buffer taken away", lambda: setattr(c.layers[3], "index_k", None)),
        ("a layer exchanged", lambda: c.layers.__setitem__(1, copy.deepcopy(c.layers[1]))),
        ("a layer in another list", lambda: setattr(c, "layers", list(c.layers[:2]) + [copy.deepcopy(c.layers[2])] + c.layers[3:])),
        ("a layer fewer", lambda: c.layers.pop()),
        ("a layer more", lambda: c.layers.append(copy.deepcopy(c.layers[2]))),
        ("a window", lambda: [setattr(lc, "window", 4) for lc in c.layers]),
    ]
    for what, step in steps:
        before = moved(c)
        step()
        now = moved(c)
        assert now == _fresh(moved, c) != before, what
    for what, step in (("a state's tensor", lambda: delattr(c.layers[4].comp_state, "kv_state")),
                       ("a buffer", lambda: delattr(c.layers[5], "win_kv"))):
        step()
        with pytest.raises(AttributeError):                       # what is missing is missed, not moved from where it was
            moved(c)
        c = _cache()
        moved(c)


def test_other_shapes_and_strides_at_the_same_address(moved):
    c = _cache()
    lc = next(lc for lc in c.layers if lc.comp_kv is not None)
    moved(c)
    lc.comp_kv.data = lc.comp_kv.data.view(4, -1, 32)             # the same bytes as twice as many rows
    assert moved(c) == _fresh(moved, c)
    lc.win_kv.data = lc.win_kv.data.view(2, -1, 64)               # half as many sequences
    with pytest.raises(ValueError, match="win_kv"):
        moved(c)
    for dense in (True, False):
        c = _cache()
        lc, pool = c.layers[0], torch.zeros(12, 8, 64, dtype=BF)
        lc.win_kv = pool[:4] if dense else pool[::2][:4]
        before = moved(c)
        lc.win_kv.data = pool[::3]                                # every third row of the pool
        assert moved(c) == _fresh(moved, c) != before
    c = _cache()
    lc = c.layers[0]
    moved(c)
    lc.win_kv.data = lc.win_kv.data.transpose(1, 2).contiguous().transpose(1, 2)
    with pytest.raises(ValueError, match="dense rows"):
        moved(c)


def test_copies_and_strangers(moved):
    c = _cache()
    moved(c)
    for other in (copy.deepcopy(c), pickle.loads(pickle.dumps(c)), copy.copy(c)):
        assert moved(other) == _fresh(moved, other)
    assert moved(copy.deepcopy(c))[0] != moved(c)[0]
    # a layer that does not count what is assigned to it: a table per call
    c.layers[1] = types.SimpleNamespace(**{k: v for k, v in vars(c.layers[1]).items() if k != "_changes"})
    moved(c)
    c.layers[1].win_kv = torch.ones_like(c.layers[1].win_kv)
    assert moved(c) == _fresh(moved, c)


def test_two_caches_are_compared_again(moved):
    from dsv41.cache import copy_sequences
    a, b = _cache(), _cache(bsz=2)
    copy_sequences(b, a, [0, 1])
    b.layers[0].win_kv = a.layers[1].win_kv[1:3]
    with pytest.raises(ValueError, match="same memory"):
        copy_sequences(b, a, [0, 1])
    b.layers[0].win_kv = torch.zeros(2, 8, 32, dtype=BF)
    with pytest.raises(ValueError, match="differ"):
        copy_sequences(b, a, [0, 1])
    with pytest.raises(ValueError, match="differ"):
        copy_sequences(_cache(cache_format="fp8"), a, [0] * 4)


def test_sequences_are_whole_numbers(moved):
    import numpy as np
    from dsv41.cache import reorder_sequences
    c = _cache()
    for order in ([1, 0], (1, 0), range(2), np.array([1, 0], np.int16), torch.tensor([1, 0]), [np.int64(1), torch.tensor(0)]):
        reorder_sequences(c, order)
        reorder_sequences(c, order, order)
    for order in ([0.9, 0], [1.0, 0], np.array([1.0, 0.0]), torch.tensor([0.5, 1]), ["1", "0"], [None, 0]):
        with pytest.raises(TypeError):
            reorder_sequences(c, order)
        with pytest.raises(TypeError):
            reorder_sequences(c, [1, 0], order)
