"""How adapter calls split their work, by sizes (host query), and a list of calls that takes every tile and every second
launch there is: tests on the GPU run that list, and a change of the plan's constants that would leave a kernel without a
test shows here."""

from __future__ import annotations

import pytest

# sequences, tokens, k, n0, n1 (0: one projection), rank0, rank1
CALLS = {
    # tile weight rows, tile rows, more than one range, x A^T apart, workgroups per CU, columns and rows of the second launch
    (32, 32, False, False, 2, 64, 4): (3, 1, 512, 8192, 512, 8, 16),
    (32, 32, False, False, 2, 64, 16): (19, 1, 1280, 32768, 0, 16, 0),
    (32, 32, True, False, 2, 64, 4): (29, 1, 1280, 320, 0, 40, 0),
    (32, 64, False, False, 2, 64, 4): (35, 1, 512, 8192, 512, 16, 24),
    (32, 64, False, False, 2, 64, 16): (61, 1, 512, 8192, 512, 8, 8),
    (32, 64, False, False, 1, 64, 4): (47, 1, 64, 32, 0, 16, 0),
    (32, 64, True, False, 1, 64, 4): (47, 1, 2048, 160, 0, 16, 0),
    (32, 96, False, False, 1, 64, 4): (65, 1, 64, 96, 0, 8, 0),
    (32, 96, True, False, 1, 64, 4): (67, 1, 1024, 512, 0, 64, 0),
    (32, 128, False, True, 2, 0, 0): (3, 333, 320, 512, 0, 32, 0),
    (32, 128, False, False, 1, 64, 4): (128, 1, 64, 32, 32, 8, 24),
    (32, 128, True, False, 1, 64, 4): (99, 1, 2048, 640, 0, 8, 0),
    (32, 128, True, False, 1, 64, 16): (115, 1, 4096, 4096, 0, 16, 0),
    (32, 128, True, False, 2, 64, 16): (43, 3, 512, 96, 256, 16, 8),
    (32, 128, True, True, 2, 64, 16): (3, 100, 1024, 160, 0, 128, 0),
    (64, 128, False, True, 2, 0, 0): (113, 1, 512, 8192, 512, 24, 8),
    (64, 128, True, False, 2, 64, 16): (67, 1, 512, 8192, 512, 16, 16),
    (64, 128, True, False, 2, 256, 16): (4, 256, 2560, 2048, 0, 8, 0),
    (64, 128, True, True, 2, 64, 16): (4, 100, 2048, 640, 0, 128, 0),
    (64, 128, True, True, 2, 256, 16): (2, 1500, 2048, 640, 0, 24, 0),
    (128, 64, False, False, 1, 64, 16): (34, 1, 1280, 32768, 0, 64, 0),
    (128, 64, False, False, 1, 256, 16): (63, 1, 1280, 32768, 0, 16, 0),
    (128, 64, True, False, 1, 64, 4): (37, 1, 4096, 4096, 0, 8, 0),
    (128, 128, False, True, 2, 0, 0): (3, 133, 512, 8192, 512, 16, 40),
    (128, 128, True, False, 2, 64, 16): (2, 333, 5120, 1280, 512, 8, 8),
    (128, 128, True, False, 2, 256, 16): (13, 100, 5120, 1280, 512, 8, 8),
    (128, 128, True, True, 2, 64, 16): (9, 74, 5120, 1280, 512, 64, 8),
    (128, 128, True, True, 2, 256, 16): (1, 4144, 5120, 512, 0, 64, 0),
    (160, 64, True, False, 1, 64, 4): (33, 1, 8192, 5120, 0, 64, 0),
    (160, 128, False, True, 2, 0, 0): (2, 4096, 2048, 640, 0, 16, 0),
    (160, 128, True, False, 2, 64, 16): (67, 1, 8192, 5120, 0, 16, 0),
    (160, 128, True, False, 2, 256, 16): (5, 400, 5120, 1280, 0, 16, 0),
    (160, 128, True, True, 2, 64, 16): (3, 333, 5120, 1280, 0, 64, 0),
    (160, 128, True, True, 2, 256, 16): (1, 2000, 5120, 1280, 0, 32, 0),
    (256, 256, False, True, 1, 0, 0): (3, 333, 1280, 32768, 0, 32, 0),
}


def plan(b, n, k, n0, n1, rank0, rank1):
    """The key of CALLS that the call takes."""
    from dsv41 import _abi
    p = _abi.adapter_linear_plan(b * n, k, n0, n1, rank0, rank1)
    return (p.tile_weight_rows, p.tile_rows, p.ranges > 1, p.first_apart, p.per_cu, p.sum_columns, p.sum_rows)


@pytest.mark.parametrize("want,call", CALLS.items(), ids=lambda v: "-".join(map(str, map(int, v))))
def test_the_calls_take_these_kernels(want, call):
    assert plan(*call) == want


def test_the_list_is_complete():
    """A sweep over sizes takes no kernel that is not on the list."""
    shapes = [(5120, 1280, 0), (5120, 1280, 512), (5120, 512, 0), (1280, 32768, 0), (8192, 5120, 0), (512, 256, 96),
              (2048, 640, 0), (256, 160, 0), (640, 96, 0), (2560, 2048, 0), (512, 8192, 512), (4096, 4096, 0), (64, 32, 0)]
    rows = [*range(1, 130), 150, 200, 300, 400, 666, 999, 1024, 1300, 2000, 3000, 4096, 4144, 8192, 30000]
    seen = {plan(r, 1, k, n0, n1, rank, 8 if n1 else 0) for r in rows for k, n0, n1 in shapes for rank in (8, 16, 32, 64, 128)}
    assert seen <= set(CALLS), seen - set(CALLS)


def test_sizes_that_no_tile_takes():
    from dsv41 import _abi
    for bad in ((0, 64, 32, 0, 8, 0), (4, 96, 32, 0, 8, 0), (4, 64, 48, 0, 8, 0), (4, 64, 32, 0, 12, 0), (4, 64, 32, 0, 136, 0)):
        with pytest.raises(ValueError, match="plan"):
            _abi.adapter_linear_plan(*bad)
