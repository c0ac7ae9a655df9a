"""Moves of sequences refuse buffers that reach into each other, on the host: workgroups of different buffers, or of
different columns of one, run in any order, so such a move would race. Checked against every byte of the rows."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

from common import RELEASE_TOY, model_args

BF = torch.bfloat16


@pytest.fixture
def moves(monkeypatch):
    """The moves on CPU caches, the C call left out."""
    from dsv41 import _abi, cache
    monkeypatch.setattr(_abi, "_gpu", lambda name, *t: None)
    monkeypatch.setattr(_abi, "_stream", lambda t: None)
    monkeypatch.setattr(_abi, "_call", lambda name, *args: None)
    return cache


def _cache(bsz=4, cap=40, offset=9):
    from dsv41.cache import ModelCache
    c = ModelCache(model_args(RELEASE_TOY), bsz, cap, BF, "cpu")
    c.offset = offset
    return c


def _refused(fn):
    with pytest.raises(ValueError, match="same memory"):
        fn()


def test_shifted_views_in_one_cache(moves):
    c = _cache()
    pool = torch.zeros(6, 8, 64, dtype=BF)
    c.layers[0].win_kv, c.layers[1].win_kv = pool[:4], pool[2:]            # rows 2 and 3 are both layers'
    _refused(lambda: moves.reorder_sequences(c, [1, 0]))
    flat = torch.zeros(2 * 4 * 8 * 64, dtype=BF)
    one = flat[:4 * 8 * 64].view(4, 8, 64)
    for shift in (1, 8 * 64 - 1, 4 * 8 * 64 - 1):                          # odd places, down to one value in common
        c.layers[0].win_kv, c.layers[1].win_kv = one, flat[shift:shift + 4 * 8 * 64].view(4, 8, 64)
        _refused(lambda: moves.reorder_sequences(c, [1, 0]))
    c.layers[1].win_kv = flat[4 * 8 * 64:].view(4, 8, 64)                  # side by side
    moves.reorder_sequences(c, [1, 0])
    pool = torch.zeros(4, 2, 8, 64, dtype=BF)                              # every sequence's layers in turn
    c.layers[0].win_kv, c.layers[1].win_kv = pool[:, 0], pool[:, 1]
    moves.reorder_sequences(c, [1, 0])
    rows = pool.view(4, 16, 64)
    c.layers[1].win_kv = rows[:, 7:15]                                     # the last row of layer 0's as well
    _refused(lambda: moves.reorder_sequences(c, [1, 0]))
    rows = torch.zeros(8, 8, 64, dtype=BF)                                 # even and odd sequences of one pool
    c.layers[0].win_kv, c.layers[1].win_kv = rows[::2], rows[1::2]
    moves.reorder_sequences(c, [1, 0])


def test_views_between_two_caches(moves):
    a, b = _cache(), _cache(bsz=2)
    moves.copy_sequences(b, a, [0, 1])
    for la, lb in zip(a.layers, b.layers):                                 # b: rows 1 and 2 of a, row for row
        for name in moves._BUFFERS:
            if getattr(la, name) is not None:
                setattr(lb, name, getattr(la, name)[1:3])
        if la.comp_state is not None:
            lb.comp_state.kv_state, lb.comp_state.score_state = la.comp_state.kv_state[1:3], la.comp_state.score_state[1:3]
    moves.copy_sequences(b, a, [0, 1])
    moves.copy_sequences(a, b, [0, 1], [3, 0])
    one = a.layers[0].win_kv[2:3]
    single = _cache(bsz=1)
    single.layers[0].win_kv = one                                          # one sequence: its rows, whatever the stride
    moves.copy_sequences(a, single, [0], [1])
    b.layers[0].win_kv, b.layers[1].win_kv = a.layers[1].win_kv[1:3], a.layers[0].win_kv[1:3]
    _refused(lambda: moves.copy_sequences(b, a, [0, 1]))                   # another layer's rows
    _refused(lambda: moves.copy_sequences(a, b, [0, 1], [3, 0]))
    b = _cache(bsz=2)
    b.layers[0].win_kv = a.layers[0].win_kv.view(-1)[32:32 + 2 * 8 * 64].view(2, 8, 64)
    _refused(lambda: moves.copy_sequences(b, a, [0, 1]))                   # the same layer's, shifted by half a row
    b.layers[0].win_kv = a.layers[0].win_kv[::2]                           # every other row: another stride
    _refused(lambda: moves.copy_sequences(b, a, [0, 1]))


@pytest.mark.parametrize("seed", range(40))
def test_against_every_byte(moves, seed):
    """Random rows in a small space: overlap exactly where some byte belongs to two rows that are not the same row of the
    same buffer."""
    rng = np.random.default_rng(seed)
    for _ in range(50):
        n, caches = int(rng.integers(1, 4)), []
        for _ in range(int(rng.integers(1, 3))):
            batch = int(rng.integers(1, 4))
            size = rng.integers(0, 9, n)
            stride = size + rng.integers(0, 30, n)
            caches.append((np.stack([rng.integers(0, 120, n), stride, size], 1).astype(np.int64), batch))
        if len(caches) == 2 and rng.random() < 0.5:            # the second as rows of the first
            (e, b0), (f, b1) = caches
            f[:, 0], f[:, 1], f[:, 2] = e[:, 0] + e[:, 1] * int(rng.integers(0, b0)), e[:, 1], e[:, 2]
        owner, clash = {}, False
        for c, (extents, batch) in enumerate(caches):
            for i, (at, stride, size) in enumerate(extents):
                step = [e[i, 1] for e, b in caches if b > 1]
                aligned = len(caches) == 2 and len(set(step)) < 2 and (
                    (caches[0][0][i, 0] - caches[1][0][i, 0]) % max(step[0] if step else caches[1][0][i, 1], 1) == 0)
                for r in range(batch):
                    first = at + r * stride
                    who = (i if aligned else (c, i), int(first)) if aligned else (c, i, r)
                    for byte in range(first, first + size):
                        clash |= owner.setdefault(byte, who) != who
        assert moves._rows_overlap(*caches) == clash, caches


def test_the_c_call_refuses_rows_closer_than_their_bytes():
    from dsv41 import _abi
    p, one = ctypes.c_void_p(4096), lambda v: (ctypes.c_int64 * 1)(v)      # noqa: E731
    ptrs = (ctypes.c_void_p * 1)(4096)
    call = lambda stride, rows: _abi.lib().dsv41_cache_move(               # noqa: E731
        ptrs, ptrs, one(16), one(stride), one(16), (ctypes.c_uint32 * 1)(0), 1, p, p, 1, 1, rows, 0, None, 0, None)
    assert call(15, 2) == -1 and call(0, 2) == -1 and call(-16, 2) == -1
    assert call(16, 2) == -4 and call(0, 1) == -4                          # taken as far as the missing workspace
