"""How 8-bit products choose their tiles: the sizes that the GPU tests run take every shape there is."""

from __future__ import annotations

from mx8_sizes import SIZES


def test_the_tested_sizes_take_every_shape():
    from dsv41 import _abi
    few = {(0, 16, 16, 8), (0, 32, 16, 2), (0, 32, 16, 8), (0, 32, 32, 4), (0, 32, 48, 8), (0, 64, 32, 8), (0, 64, 64, 8),
           (0, 64, 96, 4)}
    many = {(1, 64, 64, 1), (1, 128, 128, 1), (1, 192, 256, 1), (1, 256, 256, 1)}
    ring = {(2, 64, 64, 1), (2, 128, 64, 1), (2, 128, 128, 1), (2, 256, 128, 1), (3, 256, 256, 2), (3, 256, 256, 4)}
    plans = [_abi.linear_mx8_plan(*size) for size in SIZES]
    assert {tuple(p) for p in plans} == few | many | ring
    for shape in many | ring:                  # with a part of a pair of steps and without, and with a part of a step
        ks = {k % 256 for p, (_, k, _) in zip(plans, SIZES) if tuple(p) == shape}
        assert 0 in ks and len(ks) >= 2, (shape, ks)
        if shape[0] == 2:                      # whole steps, and a last one that lies back
            assert any(k % 128 for k in ks), (shape, ks)


def test_small_calls_take_small_tiles():
    from dsv41 import _abi
    for rows, k, n0, n1 in [(1, 5120, 1280, 512), (1, 32, 1, 0), (16, 8192, 5120, 0), (64, 32, 32, 0), (1 << 20, 32, 1, 0)]:
        plan = _abi.linear_mx8_plan(rows, k, n0, n1)
        assert plan.kernel == 0, plan              # tiles need as many rows and outputs as they are high and wide
