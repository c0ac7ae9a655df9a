"""The C call for moves of sequences on buffers of any alignment: copied rows byte for byte, emptied rows in the fill's
word, low byte first, whatever the row's length, stride and start."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fill", [0, 0xFF800000, 0xFF80FF80, 0x04030201])
@pytest.mark.parametrize("nbytes,stride,start", [(1, 1, 0), (2, 3, 1), (5, 5, 0), (7, 9, 3), (10, 10, 0), (4, 6, 2), (12, 12, 4),
                                                 (16, 16, 0), (4099, 4100, 0), (65538, 65540, 0), (65536, 65536, 1),
                                                 (200003, 200003, 0), (131072, 131072, 0)])
def test_emptied_rows_hold_the_word(gpu, nbytes, stride, start, fill):
    from dsv41 import _abi
    print(f"[bytes] bytes={nbytes} stride={stride} start={start} fill={fill:#x}", flush=True)
    rows, lead = 4, 16
    g = torch.Generator(device="cuda").manual_seed(nbytes)
    pool = torch.randint(0, 256, (lead + start + rows * stride + 64,), generator=g, device="cuda", dtype=torch.uint8)
    before = pool.cpu().numpy()
    at = lead + start
    row = lambda a, i: a[at + i * stride: at + i * stride + nbytes]          # noqa: E731
    want = before.copy()
    word = np.frombuffer(np.uint32(fill).tobytes() * (nbytes // 4 + 1), np.uint8)[:nbytes]
    row(want, 0)[:], row(want, 1)[:], row(want, 3)[:] = word, row(before, 3), word
    order = torch.tensor([-1, 3, 2, 9], dtype=torch.int32, device="cuda")
    tables = [(ctypes.c_void_p * 1)(pool.data_ptr() + at), (ctypes.c_int64 * 1)(stride), (ctypes.c_int64 * 1)(nbytes),
              (ctypes.c_uint32 * 1)(fill)]
    ptr, step, size, word = (ctypes.addressof(t) for t in tables)
    need = _abi.cache_move_workspace_bytes(1, 4)
    ws = torch.empty(need, dtype=torch.uint8, device="cuda")
    _abi._call("dsv41_cache_move", ptr, ptr, step, step, size, word, 1, order.data_ptr(), None, 4, rows, rows, 1,
               ws.data_ptr(), need, _abi._stream(order))
    assert np.array_equal(pool.cpu().numpy(), want)
