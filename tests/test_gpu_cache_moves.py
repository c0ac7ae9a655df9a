"""Sequences forked, admitted, moved and emptied in the caches: bytes against indexing on the host."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from common import C1, C4_TOY, RELEASE_TOY, SEED_BASE, args, load_stack, model_args
from oracle import cpu_ref as R

pytestmark = pytest.mark.gpu

FORMATS = [("dense", "dense", 1), ("mxfp4", "dense", 1), ("dense", "fp8", 1), ("dense", "fp8", 32), ("mxfp4", "fp4", 1),
           ("mxfp4", "packed", 1)]


def _tensors(cache):
    from dsv41.cache import _BUFFERS
    for i, lc in enumerate(cache.layers):
        for name in _BUFFERS:
            if getattr(lc, name) is not None:
                yield i, lc, name, getattr(lc, name)
        if lc.comp_state is not None:
            yield i, lc, "kv_state", lc.comp_state.kv_state
            yield i, lc, "score_state", lc.comp_state.score_state


def _cache(cfg, bsz, cap, offset, fmt, seed, dtype=torch.bfloat16):
    """A cache of random bytes (NaN patterns among them) at a position."""
    from dsv41.cache import ModelCache
    index, form, rb = fmt
    cache = ModelCache(model_args(cfg), bsz, cap, dtype, "cuda", index, form, rb)
    g = torch.Generator(device="cuda").manual_seed(SEED_BASE + seed)
    for *_, t in _tensors(cache):
        t.view(torch.uint8).random_(0, 256, generator=g)
    cache.offset = offset
    return cache


def _bytes(cache):
    return [t.view(torch.uint8).cpu().numpy().copy() for *_, t in _tensors(cache)]


def _visible(lc, name, offset):
    if name in ("win_kv", "win_kv8"):
        return min(offset, lc.window)
    if name in ("kv_state", "score_state"):
        return lc.ratio
    n = offset // lc.ratio
    return -(-n // lc.fp8_rb) if name in ("comp_ks", "index_k8s") else n


def _expect(dst, src, offset, order, rows):
    """dst's bytes after the moves, from both caches' bytes before them."""
    ours, theirs = _bytes(dst), _bytes(src)
    for (_, lc, name, _), new, old in zip(_tensors(dst), ours, theirs):
        v, was = _visible(lc, name, offset), old.copy()
        for s, d in zip(order, rows):
            if not 0 <= d < new.shape[0]:
                continue
            if 0 <= s < old.shape[0]:
                new[d, :v] = was[s, :v]
            else:
                new[d, :v] = np.tile(np.array([0, 0, 128, 255], np.uint8), new.shape[2] // 4) if name == "score_state" else 0
    return ours


def _same(cache, want):
    for (i, _, name, t), w in zip(_tensors(cache), want):
        got = t.view(torch.uint8).cpu().numpy()
        assert np.array_equal(got, w), (i, name, np.argwhere((got != w).any(axis=-1))[:5].tolist())


def _dev(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("fmt", FORMATS, ids=lambda f: f"{f[0]}-{f[1]}-{f[2]}")
@pytest.mark.parametrize("offset", [0, 1, 3, 7, 33, 60])
def test_reorder_in_place(gpu, fmt, offset):
    """Permutations with cycles, forks, emptied rows and rows left alone, over the ratios 1 and 2 of the release's
    topology, a window that has and has not wrapped, groups open and closed, row bytes of every alignment."""
    from dsv41.cache import reorder_sequences
    cfg = dict(RELEASE_TOY, head_dim=512) if fmt[1] in ("fp4", "packed") else RELEASE_TOY
    for seed, order in enumerate([[4, 3, 2, 1, 0], [1, 2, 3, 4, 0], [2, 2, 2, 2, 2], [0, 1, 2, 3, 4], [-1, 0, -1, 9, 1],
                                  [3], [-5, 1 << 30]]):
        print(f"[moves] {fmt} offset={offset} order={order}", flush=True)
        cache = _cache(cfg, 5, 61, offset, fmt, seed)
        want = _expect(cache, cache, offset, order, range(len(order)))
        reorder_sequences(cache, _dev(order))
        _same(cache, want)
        assert cache.offset == offset


@pytest.mark.parametrize("fmt", FORMATS, ids=lambda f: f"{f[0]}-{f[1]}-{f[2]}")
def test_rows_and_repeats(gpu, fmt):
    """Named destinations: outside ones move nothing, of several to one row the last counts; host sequences and device
    tensors alike."""
    from dsv41.cache import reorder_sequences
    cfg = dict(C4_TOY, head_dim=512) if fmt[1] in ("fp4", "packed") else C4_TOY
    for seed, (order, rows) in enumerate([([0, 1, 2], [5, 0, 1]), ([4, -1], [0, 4]), ([1, 2, 3, -1, 5], [0, 0, 0, 2, 2]),
                                          ([3, 0], [-1, 6]), ([2, 1], [2, 1])]):
        cache = _cache(cfg, 6, 50, 41, fmt, seed)
        want = _expect(cache, cache, 41, order, rows)
        reorder_sequences(cache, _dev(order), _dev(rows))
        _same(cache, want)
        if all(0 <= d < 6 for d in rows):
            again = _cache(cfg, 6, 50, 41, fmt, seed)
            reorder_sequences(again, order, rows)
            _same(again, want)
    cache = _cache(cfg, 6, 50, 41, fmt, 9)
    want = _bytes(cache)
    reorder_sequences(cache, [], [])
    reorder_sequences(cache, _dev([]))
    _same(cache, want)


@pytest.mark.parametrize("bsz", [17, 64, 300])
def test_many_rows(gpu, bsz):
    """More moves than a pass holds whole spans of: random maps of every row."""
    from dsv41.cache import reorder_sequences
    rng = np.random.default_rng(bsz)
    for seed in range(3):
        order = rng.integers(-1, bsz, bsz).tolist() if seed else rng.permutation(bsz).tolist()
        cache = _cache(dict(RELEASE_TOY, window_size=40), bsz, 150, 131, ("dense", "dense", 1), seed)
        want = _expect(cache, cache, 131, order, range(bsz))
        reorder_sequences(cache, _dev(order))
        _same(cache, want)


@pytest.mark.parametrize("fmt", FORMATS, ids=lambda f: f"{f[0]}-{f[1]}-{f[2]}")
def test_copy_between_caches(gpu, fmt):
    """A prompt forked into a fresh batch of another capacity, and one sequence admitted into a running one."""
    from dsv41.cache import copy_sequences
    cfg = dict(RELEASE_TOY, head_dim=512) if fmt[1] in ("fp4", "packed") else RELEASE_TOY
    src = _cache(cfg, 2, 45, 37, fmt, 1)
    dst = _cache(cfg, 4, 100, 0, fmt, 2)
    want, before = _expect(dst, src, 37, [1, 1, 0, 1], range(4)), _bytes(src)
    copy_sequences(dst, src, [1, 1, 0, 1])
    _same(dst, want)
    assert dst.offset == 37
    want = _expect(dst, src, 37, [0], [2])
    copy_sequences(dst, src, _dev([0]), _dev([2]))
    _same(dst, want)
    _same(src, before)
    src.offset = 38
    with pytest.raises(ValueError, match="single rows"):
        copy_sequences(dst, src, [0], [2])
    with pytest.raises(ValueError, match="into a cache of 4"):
        copy_sequences(dst, src, [0] * 5)
    with pytest.raises(ValueError, match="must lie in"):
        copy_sequences(dst, src, [2] * 4)
    with pytest.raises(ValueError, match="must lie in"):
        copy_sequences(dst, src, [0], [4])
    small = _cache(cfg, 4, 30, 0, fmt, 3)
    with pytest.raises(ValueError, match="holds"):
        copy_sequences(small, src, [0] * 4)
    other = _cache(dict(cfg, n_layers=6, compress_ratios=cfg["compress_ratios"][:6], index_source_layers=(2, 5)), 4, 100,
                   0, fmt, 3)
    with pytest.raises(ValueError, match="differ"):
        copy_sequences(other, src, [0] * 4)
    assert dst.offset == 37
    _same(dst, want)


def test_strided_buffers_and_many_layers(gpu):
    """Buffers that are views of a larger batch, and more of them than one launch takes."""
    from dsv41.cache import reorder_sequences
    cfg = dict(C4_TOY, n_layers=90, compress_ratios=(4,) * 90, kv_source_layers=tuple(range(0, 90, 9)),
               index_source_layers=tuple(range(0, 90, 9)), candidate_source_layer=-1)
    cache = _cache(cfg, 6, 30, 29, ("dense", "dense", 1), 4)
    for lc in cache.layers:
        lc.win_kv = lc.win_kv[::2]
        if lc.comp_kv is not None:
            lc.comp_kv, lc.index_k = lc.comp_kv[1::2], lc.index_k[:3]
            lc.comp_state.kv_state, lc.comp_state.score_state = lc.comp_state.kv_state[:3], lc.comp_state.score_state[3:]
    want = _expect(cache, cache, 29, [2, 0, 1], range(3))
    reorder_sequences(cache, _dev([2, 0, 1]))
    _same(cache, want)


def test_replaced_buffers_are_seen(gpu):
    """Every call looks at the buffers as they are: ones replaced whole, states replaced, layers replaced, contents moved
    to other storage; copies and pickles of a cache that has moved sequences work."""
    import copy
    import pickle

    from dsv41.cache import reorder_sequences
    from dsv41.compressor import CompressorState
    cache = _cache(RELEASE_TOY, 3, 30, 19, ("dense", "dense", 1), 8)
    order = _dev([1, 2, 0])

    def moves():
        want = _expect(cache, cache, 19, [1, 2, 0], range(3))
        reorder_sequences(cache, order)
        _same(cache, want)

    moves()
    owner = next(lc for lc in cache.layers if lc.comp_state is not None)
    owner.comp_kv = owner.comp_kv.clone().mul_(2)
    moves()
    owner.comp_state = CompressorState(3, owner.ratio, 64)
    owner.comp_state.kv_state.normal_()
    moves()
    owner.win_kv.data = owner.win_kv.clone()
    moves()
    cache.layers[0] = _cache(RELEASE_TOY, 3, 30, 19, ("dense", "dense", 1), 9).layers[0]
    moves()
    other = copy.deepcopy(cache)
    assert len(pickle.dumps(cache)) > 0
    before = _bytes(cache)
    reorder_sequences(other, order)
    _same(cache, before)
    _same(other, _expect(cache, cache, 19, [1, 2, 0], range(3)))
    owner.win_kv = owner.win_kv[:2]
    with pytest.raises(ValueError, match="win_kv"):
        reorder_sequences(cache, order)


def test_two_streams_at_once(gpu):
    """Calls on two streams have workspaces of their own."""
    from dsv41.cache import reorder_sequences
    caches = [_cache(C4_TOY, 6, 60, 50, ("dense", "dense", 1), 10 + i) for i in range(2)]
    orders = [[5, 4, 3, 2, 1, 0], [1, -1, 0, 5, 5, 2]]
    wants = [_expect(c, c, 50, o, range(6)) for c, o in zip(caches, orders)]
    devs = [_dev(o) for o in orders]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for s, c, o in zip(streams, caches, devs):
        with torch.cuda.stream(s):
            reorder_sequences(c, o)
    torch.cuda.synchronize()
    for c, w in zip(caches, wants):
        _same(c, w)


def test_captured_moves_follow_the_order(gpu):
    from dsv41.cache import reorder_sequences
    cache = _cache(RELEASE_TOY, 4, 40, 37, ("dense", "dense", 1), 5)
    order = _dev([0, 1, 2, 3])
    reorder_sequences(cache, order)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        reorder_sequences(cache, order)
    for o in ([1, 0, 3, 2], [3, 3, 0, 1], [0, -1, 2, 2], [1, 2, 3, 0]):
        order.copy_(_dev(o))
        want = _expect(cache, cache, 37, o, range(4))
        graph.replay()
        torch.cuda.synchronize()
        _same(cache, want)


def test_offsets_past_32_bits(gpu):
    """Rows of 1.6 GB, the last one past 4 GB of its buffer: two swapped, one emptied."""
    from dsv41.cache import reorder_sequences
    cfg = dict(C1, n_layers=1, head_dim=512, compress_ratios=(1,), kv_source_layers=(0,), index_source_layers=())
    cache = _cache(cfg, 4, 1600000, 1599999, ("dense", "dense", 1), 11)
    kv = cache.layers[0].comp_kv
    assert kv.stride(0) * 2 * 3 > 1 << 32
    old = [kv[i].clone() for i in range(4)]
    reorder_sequences(cache, _dev([3, -1, 2, 0]))
    seen = 1599999
    same = lambda a, b: torch.equal(a.view(torch.int16), b.view(torch.int16))     # noqa: E731
    assert same(kv[0, :seen], old[3][:seen]) and same(kv[2], old[2]) and same(kv[3, :seen], old[0][:seen])
    assert not kv[1, :seen].view(torch.int16).any()
    assert all(same(kv[i, seen:], old[i][seen:]) for i in range(4))


def test_engram_ids_move_too(gpu):
    from dsv41.cache import copy_sequences, reorder_sequences
    cfg = dict(RELEASE_TOY, engram_layer_ids=(1,))
    a = _cache(cfg, 3, 40, 21, ("dense", "dense", 1), 6)
    a.engram_ids[...] = np.arange(3 * 40).reshape(3, 40)
    want = a.engram_ids.copy()
    want[:, :21] = want[[2, 0, 0], :21]
    want[1, :21] = 0
    reorder_sequences(a, _dev([2, -1, 0]))
    assert np.array_equal(a.engram_ids, want)
    b = _cache(cfg, 2, 64, 0, ("dense", "dense", 1), 7)
    copy_sequences(b, a, [2, 0])
    assert np.array_equal(b.engram_ids[:, :21], want[[2, 0], :21])
    c = _cache(RELEASE_TOY, 2, 64, 0, ("dense", "dense", 1), 7)
    with pytest.raises(ValueError, match="engram"):
        copy_sequences(c, a, [0, 0])


def test_serving_run_with_forks_adapters_and_compaction(gpu, monkeypatch):
    """One prompt computed once, forked into a batch whose sequences go on under their own adapters, beams that follow a
    survivor, finished rows filled from the end: against the same tokens run through a batch that never moved. The
    float32 stack agrees with itself to 1e-5 whatever the batch."""
    import dsv41.fakequant as FQ
    from dsv41.cache import copy_sequences, reorder_sequences
    from dsv41.model import AttentionStack
    monkeypatch.setattr(FQ, "DISABLE", True)
    st = AttentionStack(model_args(C1), torch.float32, gpu)
    load_stack(st, R.make_params(args(C1), SEED_BASE, "f32"))
    g = torch.Generator(device="cuda").manual_seed(SEED_BASE)
    for banks in st.add_adapters(3, 8):
        for bank in banks.values():
            for t in range(3):
                bank.load(t, torch.randn(8, bank.in_features, generator=g, device="cuda") * bank.in_features ** -0.5,
                          torch.randn(bank.out_features, 8, generator=g, device="cuda") * 0.02, 1.0)
    prompt = torch.randn(1, 37, C1["dim"], generator=g, device="cuda")
    tokens = [torch.randn(4, 1, C1["dim"], generator=g, device="cuda") for _ in range(8)]

    def close(a, b):
        assert (a - b).abs().max() <= 1e-5 * max(1.0, float(b.abs().max()))

    one = st.make_cache(1, 64)
    base = torch.tensor([-1], dtype=torch.int32, device="cuda")
    st(prompt, one, base)
    batch = st.make_cache(4, 64)
    copy_sequences(batch, one, [0] * 4)
    assert batch.offset == 37
    still = st.make_cache(4, 64)
    st(prompt.expand(4, -1, -1).contiguous(), still, base.expand(4).contiguous())
    ids = torch.tensor([0, -1, 2, 1], dtype=torch.int32, device="cuda")
    for t in tokens[:3]:
        close(st(t, batch, ids), st(t, still, ids))
    # every sequence becomes another one, adapters and tokens with it
    order = torch.tensor([2, 0, 3, 1], dtype=torch.int32, device="cuda")
    reorder_sequences(batch, order)
    p = order.long()
    for t in tokens[3:5]:
        close(st(t[p].contiguous(), batch, ids[p].contiguous()), st(t, still, ids)[p])
    # row 1 (sequence 0) has finished: the last row (sequence 1) takes its place, three go on
    reorder_sequences(batch, [3, -1], [1, 3])
    live = torch.tensor([2, 1, 3], device="cuda")
    for t in tokens[5:]:
        close(st(t[live].contiguous(), batch, ids[live].contiguous()), st(t, still, ids)[live])
    assert all(not lc.comp_kv[3].any() for lc in batch.layers if lc.comp_kv is not None)
