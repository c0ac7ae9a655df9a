"""Incremental attention state in HBM (deepseek_v41_mlx/cache.py:27-78).

Per layer:

* ``win_kv`` -- every layer: a ring of ``window_size`` KV rows, position p at slot p % window;
* ``comp_kv`` -- kv-source (owner) layers only: one latent per completed group, append-only;
  consumer layers never copy it: they read the most recent owner's buffer in place through
  ``SharedState.kv_src_cache``;
* ``comp_state`` -- ratio > 1 owners: the fp32 kv/score rows of the open group;
* ``index_k`` -- owners that are also index sources: the indexer's key cache, read in place
  by every index source below them. With ``index_format="mxfp4"`` the keys -- fp4
  fake-quantized by construction (indexer.py:100-104) -- are held losslessly packed instead:
  ``index_k4`` (e2m1 codes, [b, n, Di/2] bytes) and ``index_ks`` (ue8m0 block scales,
  [b, n, Di/32] bytes), and ``index_k`` is None.

``cache_format="fp8"`` is the fp8 cache variant: the compressed KV and the index keys are
stored as e4m3fn codes with one ue8m0 scale byte per 32 channels of each row (``comp_kv8`` /
``comp_ks``, ``index_k8`` / ``index_k8s``; ``comp_kv`` and ``index_k`` are None), written with
fake_quant_fp8_ue8m0's formula in place of the reference's fp4 QAT at those two stores and
dequantized in-kernel. The window ring stays in ``dtype``.

``cache_format="fp4"`` holds the compressed KV -- fp4/e4m3 fake-quantized by construction
(attention.py:157-163) -- losslessly packed: ``comp_kv4``, rows of d/2 bytes of e2m1 codes then
d/16 e4m3 scale bytes (288 bytes for 512 channels; ``comp_kv`` is None). The index keys follow
``index_format`` (MXFP4 is their lossless packed form), the window ring stays in ``dtype``.
``cache_format="packed"`` adds the window ring in its lossless packed form: ``win_kv8``, MXFP8
rows of d e4m3fn codes then d/32 ue8m0 scale bytes (528 bytes for 512 channels; ``win_kv`` is
None), for window KV that carries the fp8 QAT of attention.py:120-122. The packed stores encode
their QAT, so with the QAT switched off they quantize at the store.

All buffers are plain torch device tensors with the reference's attribute names. The kernels
update them in place, so a snapshot must copy: ``lc.win_kv[:]`` -- which in MLX pins the
pre-step value (generate.py:18-44) -- is a view in torch. ``snapshot(cache)`` and
``restore(cache, snap)`` are the torch counterparts of generate.py's ``_cache_snapshot`` /
``_cache_restore``: they copy every buffer of every format, and restore writes back into the
same tensors, so references to them (a captured HIP graph, a consumer's view) stay valid.

``dtype`` defaults to fp32, the reference's default (cache.py:29, 72). The attention layer
converts at every boundary of a cache held in another dtype than its activations, as the
reference does (attention.py:127, 163, 166); a cache in the activation dtype is read in place.
"""

from __future__ import annotations

import ctypes
import operator
import weakref

import numpy as np
import torch

from . import _abi
from .compressor import CompressorState, CountedAttributes
from .config import ModelArgs


INDEX_FORMATS = ("dense", "mxfp4")
CACHE_FORMATS = ("dense", "fp8", "fp4", "packed")


class PackedKeys:
    """Index keys of a packed cache as the indexer takes them: kind "mxfp4" or "fp8", the code
    and scale views of rows [:bsz, :n], and the rows one scale byte covers (rb: 1, or 32 for an
    fp8 cache of 32 x 32 blocks)."""

    def __init__(self, kind: str, codes: torch.Tensor, scales: torch.Tensor, rb: int = 1):
        self.kind, self.codes, self.scales, self.rb = kind, codes, scales, rb

    @property
    def shape(self):
        return self.codes.shape


class LayerCache(CountedAttributes):
    def __init__(self, bsz: int, args: ModelArgs, layer_id: int, max_seq_len: int,
                 dtype=torch.float32, device="cuda", index_format: str = "dense", cache_format: str = "dense",
                 fp8_block_rows: int = 1):
        if index_format not in INDEX_FORMATS:
            raise ValueError(f"index_format must be one of {INDEX_FORMATS}, got {index_format!r}")
        if cache_format not in CACHE_FORMATS:
            raise ValueError(f"cache_format must be one of {CACHE_FORMATS}, got {cache_format!r}")
        if fp8_block_rows not in (1, 32):
            raise ValueError(f"fp8_block_rows must be 1 or 32, got {fp8_block_rows}")
        fp8 = cache_format == "fp8"
        # fp8 caches: one ue8m0 scale byte per 32 channels of every fp8_rb rows (32: 32 x 32 blocks)
        self.fp8_rb = fp8_block_rows if fp8 else 1
        self.window = args.window_size
        self.ratio = args.compress_ratio(layer_id)
        self.is_kv_source = layer_id in args.kv_source_layers
        self.dtype = dtype
        self.win_kv = self.win_kv8 = None
        if cache_format == "packed":
            self.win_kv8 = torch.zeros(bsz, self.window, _abi.mxfp8_row_bytes(args.head_dim), dtype=torch.uint8,
                                       device=device)
        else:
            self.win_kv = torch.zeros(bsz, self.window, args.head_dim, dtype=dtype, device=device)
        self.comp_kv = None
        self.comp_state = None
        self.index_k = None
        self.index_k4 = None
        self.index_ks = None
        self.comp_kv8 = self.comp_ks = self.index_k8 = self.index_k8s = None
        self.comp_kv4 = None
        if self.is_kv_source:
            n_comp = max_seq_len // self.ratio
            d = args.head_dim
            n_blk = -(-n_comp // self.fp8_rb)
            if fp8:
                self.comp_kv8 = torch.zeros(bsz, n_comp, d, dtype=torch.uint8, device=device)
                self.comp_ks = torch.zeros(bsz, n_blk, d // 32, dtype=torch.uint8, device=device)
            elif cache_format in ("fp4", "packed"):
                self.comp_kv4 = torch.zeros(bsz, n_comp, _abi.fp4_row_bytes(d), dtype=torch.uint8, device=device)
            else:
                self.comp_kv = torch.zeros(bsz, n_comp, d, dtype=dtype, device=device)
            if self.ratio > 1:
                self.comp_state = CompressorState(bsz, self.ratio, args.head_dim, device)
            if layer_id in args.index_source_layers:
                di = args.index_head_dim
                if fp8:
                    self.index_k8 = torch.zeros(bsz, n_comp, di, dtype=torch.uint8, device=device)
                    self.index_k8s = torch.zeros(bsz, n_blk, di // 32, dtype=torch.uint8, device=device)
                elif index_format == "mxfp4":
                    self.index_k4 = torch.zeros(bsz, n_comp, di // 2, dtype=torch.uint8, device=device)
                    self.index_ks = torch.zeros(bsz, n_comp, di // 32, dtype=torch.uint8, device=device)
                else:
                    self.index_k = torch.zeros(bsz, n_comp, di, dtype=dtype, device=device)

    def index_keys(self, bsz: int, n: int):
        """The first n keys of rows [:bsz] in the form the indexer takes: a dense view, or the
        PackedKeys of an MXFP4 or fp8 cache."""
        if self.index_k4 is not None:
            return PackedKeys("mxfp4", self.index_k4[:bsz, :n], self.index_ks[:bsz, :n])
        if self.index_k8 is not None:
            return PackedKeys("fp8", self.index_k8[:bsz, :n], self.index_k8s[:bsz, :-(-n // self.fp8_rb)], self.fp8_rb)
        return self.index_k[:bsz, :n]

    def comp_source(self, bsz: int):
        """The compressed cache of rows [:bsz] as the attention reads it: (kind, tensor), kind
        "dense", "fp8" (codes; the scales are ``comp_ks``) or "fp4" (packed rows)."""
        if self.comp_kv8 is not None:
            return "fp8", self.comp_kv8[:bsz]
        if self.comp_kv4 is not None:
            return "fp4", self.comp_kv4[:bsz]
        return "dense", self.comp_kv[:bsz]

    def ring(self):
        """The window ring as the attention reads it: (kind, tensor), kind "dense" or "mxfp8"."""
        return ("mxfp8", self.win_kv8) if self.win_kv8 is not None else ("dense", self.win_kv)

    def window_chrono(self, pos: int) -> torch.Tensor:
        """The ring in chronological order: positions [pos - Wp, pos), Wp = min(pos, window).
        Rows of the packed ring come back as their uint8 MXFP8 rows."""
        w = self.window
        if self.win_kv8 is not None:
            wp = min(pos, w)
            slots = (torch.arange(wp, device=self.win_kv8.device) + (pos - wp)) % w
            return self.win_kv8[:, slots]
        wp = min(pos, w)
        slots = (torch.arange(wp, device=self.win_kv.device) + (pos - wp)) % w
        return self.win_kv[:, slots]

    def write_window(self, pos: int, kv: torch.Tensor) -> None:
        """Write chunk KV at positions [pos, pos+n) into the ring (cache.py:61-67)."""
        if self.win_kv8 is not None:
            _abi.window_write_mxfp8(self.win_kv8, kv.to(self.dtype).contiguous(), pos)
        else:
            _abi.window_write(self.win_kv, kv.to(self.dtype).contiguous(), pos)


class ModelCache:
    def __init__(self, args: ModelArgs, bsz: int = 1, max_seq_len: int | None = None,
                 dtype=torch.float32, device="cuda", index_format: str = "dense", cache_format: str = "dense",
                 fp8_block_rows: int = 1):
        self.max_seq_len = max_seq_len or min(args.max_seq_len, 4096)
        self.offset = 0
        self.layers = [LayerCache(bsz, args, i, self.max_seq_len, dtype, device, index_format, cache_format,
                                  fp8_block_rows)
                       for i in range(args.n_layers)]
        # token ids the engram hasher reads back (cache.py:77-78); host memory, as there
        self.engram_ids = (np.zeros((bsz, self.max_seq_len), dtype=np.int64)
                           if args.engram_layer_ids else None)


_BUFFERS = ("win_kv", "comp_kv", "index_k", "index_k4", "index_ks", "comp_kv8", "comp_ks", "index_k8", "index_k8s",
            "comp_kv4", "win_kv8")


def snapshot(cache: ModelCache):
    """Copies of every cache buffer and the offset (generate.py:18-30 takes the same state)."""
    layers = []
    for lc in cache.layers:
        bufs = {name: getattr(lc, name).clone() for name in _BUFFERS if getattr(lc, name) is not None}
        cs = lc.comp_state
        state = (cs.kv_state.clone(), cs.score_state.clone()) if cs is not None else None
        layers.append((bufs, state))
    eng = cache.engram_ids.copy() if cache.engram_ids is not None else None
    return cache.offset, layers, eng


def restore(cache: ModelCache, snap) -> None:
    """Write a snapshot back (generate.py:33-44), into the same tensors."""
    offset, layers, eng = snap
    if len(layers) != len(cache.layers):
        raise ValueError(f"snapshot of {len(layers)} layers for a cache of {len(cache.layers)}")
    cache.offset = offset
    for lc, (bufs, state) in zip(cache.layers, layers):
        for name, t in bufs.items():
            getattr(lc, name).copy_(t)
        if state is not None:
            lc.comp_state.kv_state.copy_(state[0])
            lc.comp_state.score_state.copy_(state[1])
    if eng is not None:
        cache.engram_ids[...] = eng


# ---------------------------------------------------------------------------- sequences of a batch

_MINUS_INF = 0xFF800000


def _rows_overlap(*caches) -> bool:
    """Whether two rows (start, bytes between rows, bytes of a row; rows of one cache or of two) have bytes in common.
    Of two caches, buffer i of the one may be whole rows of buffer i of the other, row for row: a move reads all rows of a
    buffer before it writes any, but different buffers, or different columns of one, at any time. Rows of one pool in
    turn (views whose spans interlace) are apart."""
    starts, ends, buffers = [], [], []
    for extents, batch in caches:
        at, stride, size = extents.T
        starts.append(at)
        ends.append(at + stride * (batch - 1) + size)
    lo, hi = np.concatenate(starts), np.concatenate(ends)
    order = np.argsort(lo)
    if (lo[order][1:] >= np.maximum.accumulate(hi[order])[:-1]).all():
        return False                       # not even the buffers' whole spans meet
    starts, ends = [], []
    n = len(caches[0][0])
    aligned = np.ones(n, dtype=bool)
    if len(caches) == 2:
        (a, batch_a), (b, batch_b) = caches
        step = a[:, 1] if batch_a > 1 else b[:, 1]
        aligned = ((a[:, 0] - b[:, 0]) % np.maximum(step, 1) == 0) & (
            (a[:, 1] == b[:, 1]) if batch_a > 1 and batch_b > 1 else True)
    for i, (extents, batch) in enumerate(caches):
        at, stride, size = extents.T
        first = at[:, None] + stride[:, None] * np.arange(batch)
        starts.append(first.ravel())
        ends.append((first + size[:, None]).ravel())
        buffers.append(np.repeat(np.where(aligned, np.arange(n), np.arange(n) + n * i), batch))
    lo, hi, buffer = np.concatenate(starts), np.concatenate(ends), np.concatenate(buffers)
    held = hi > lo
    lo, hi, buffer = lo[held], hi[held], buffer[held]
    order = np.lexsort((hi, buffer, lo))
    lo, hi, buffer = lo[order], hi[order], buffer[order]
    met = lo[1:] < np.maximum.accumulate(hi)[:-1]
    return bool((met & ((lo[1:] != lo[:-1]) | (buffer[1:] != buffer[:-1]))).any())


_changes = operator.attrgetter("_changes")


class _RowTable:
    """A cache's buffers as moves of sequences take them: one entry per buffer, in layer order. Kept on the ModelCache
    (it holds no buffer alive, and copies and pickles of the cache leave it out) and built again when a layer or a state
    is another one, when anything has been assigned to one of them (a buffer exchanged, added or taken away), and when a
    buffer lies elsewhere or has another shape or other strides."""

    def __init__(self, cache: ModelCache):
        self.layout, self.width, tensors, fills = [], [], [], []
        counted = []                       # layers and states
        self.kinds, self.need = {}, []     # (what the rows count, ratio, rows per scale), the fewest rows of such a buffer
        self.kind = []                     # a buffer's entry of those
        for i, lc in enumerate(cache.layers):
            names = [n for n in _BUFFERS if getattr(lc, n) is not None]
            if lc.comp_state is not None:
                names += ["comp_state.kv_state", "comp_state.score_state"]
                counted.append(lc.comp_state)
            for name in names:
                t = operator.attrgetter(name)(lc)
                if t.dim() != 3 or t.stride(2) != 1 or t.stride(1) != t.shape[2] or (
                        t.shape[0] > 1 and t.stride(0) < t.shape[1] * t.shape[2]):
                    raise ValueError(f"layer {i}: {name} {tuple(t.shape)} must be [sequences, rows, channels] with dense rows")
                kind = ("state", t.shape[1], 1) if name.endswith("_state") else ("ring", lc.window, 1) if name.startswith(
                    "win") else ("comp", lc.ratio, lc.fp8_rb if name in ("comp_ks", "index_k8s") else 1)
                if kind not in self.kinds:
                    self.kinds[kind] = len(self.need)
                    self.need.append(t.shape[1])
                k = self.kinds[kind]
                tensors.append(t)
                self.layout.append((i, name, t.dtype, t.shape[2], kind))
                self.kind.append(k)
                self.width.append(t.shape[2] * t.element_size())
                self.need[k] = min(self.need[k], t.shape[1])
                fills.append(_MINUS_INF if name.endswith("score_state") else 0)
        if not tensors:
            raise ValueError("a cache without buffers")
        self.batch, self.device = tensors[0].shape[0], tensors[0].device
        for (i, name, *_), t in zip(self.layout, tensors):
            if t.shape[0] != self.batch or t.device != self.device:
                raise ValueError(f"layer {i}: {name} {tuple(t.shape)} on {t.device} in a cache of {self.batch} sequences on "
                                 f"{self.device}")
        counted[:0] = cache.layers
        # an object that does not count its changes is not trusted to have had none: the table serves one call
        self.known = all(isinstance(c, CountedAttributes) for c in counted)
        self.layers, self.counted = len(cache.layers), [weakref.ref(c) for c in counted] if self.known else []
        self.changes = [c._changes for c in counted] if self.known else None
        self.tensors = [weakref.ref(t) for t in tensors]
        self.where = [t.data_ptr() for t in tensors]
        self.shapes, self.steps = [t.size() for t in tensors], [t.stride() for t in tensors]
        self.dense = all(t.is_contiguous() for t in tensors)
        n = len(tensors)
        # where the buffers' rows lie: first row, bytes between rows, bytes of a row
        self.extents = np.array([(t.data_ptr(), t.stride(0) * t.element_size(), t.shape[1] * w)
                                 for t, w in zip(tensors, self.width)], dtype=np.int64)
        self.partners = weakref.WeakSet()  # other caches' tables that go with this one (_pair)
        if _rows_overlap((self.extents, self.batch)):
            raise ValueError("two buffers of the cache lie in the same memory")
        self.kind, self.width = np.array(self.kind), np.array(self.width, dtype=np.int64)
        self.words = ctypes.c_int64 * n
        self.pointers = self.words(*self.where)
        self.strides = self.words(*(t.stride(0) * t.element_size() for t in tensors))
        self.fills = (ctypes.c_uint32 * n)(*fills)

    def __reduce__(self):
        return type(None), ()

    def current(self, cache: ModelCache) -> bool:
        if not self.known:
            return False
        counted, now = [r() for r in self.counted], [r() for r in self.tensors]
        try:
            return (counted[:self.layers] == list(cache.layers)
                    and list(map(_changes, counted)) == self.changes
                    and list(map(torch.Tensor.data_ptr, now)) == self.where
                    and list(map(torch.Tensor.size, now)) == self.shapes
                    # a shape without gaps has one set of strides (2.0 us for 56 buffers, their strides 3.3)
                    and (self.dense and all(map(torch.Tensor.is_contiguous, now))
                         or list(map(torch.Tensor.stride, now)) == self.steps))
        except (AttributeError, TypeError):    # a state or a buffer has gone
            return False

    def check(self, offset: int) -> list:
        """Rows that `offset` positions have written, by kind of buffer: ring slots, compressed rows (or their scale
        blocks), the open group's state."""
        rows = []
        for (what, per, block), held in zip(self.kinds, self.need):
            n = per if what == "state" else min(offset, per) if what == "ring" else -(-(offset // per) // block)
            if n > held:
                raise ValueError(f"a buffer holds {held} of the {n} rows that {offset} positions take")
            rows.append(n)
        return rows

    def visible(self, offset: int):
        """Bytes of a sequence that move, buffer by buffer."""
        rows = self.check(offset)
        return self.words.from_buffer(np.array(rows, dtype=np.int64)[self.kind] * self.width)


def _row_table(cache: ModelCache) -> _RowTable:
    table = cache.__dict__.get("_row_table")
    if table is None or not table.current(cache):
        table = cache._row_table = _RowTable(cache)
    return table


def _pair(what: str, ours: _RowTable, theirs: _RowTable) -> None:
    """What two caches' buffers must have in common, and apart, for sequences to move between them: once per pair."""
    if ours.layout != theirs.layout:
        raise ValueError(f"{what}: the caches differ in layers, formats, widths or ratios")
    if ours.device != theirs.device:
        raise ValueError(f"{what}: caches on {ours.device} and {theirs.device}")
    if _rows_overlap((ours.extents, ours.batch), (theirs.extents, theirs.batch)):
        raise ValueError(f"{what}: buffers of the caches lie in the same memory")
    ours.partners.add(theirs)


def _index(what: str, values, rows: int, low: int, device) -> torch.Tensor:
    """order or rows as an int32 device vector; entries of a host sequence are checked here, those of a device tensor
    by the kernel."""
    if isinstance(values, torch.Tensor) and values.is_cuda:
        return values
    values = [operator.index(v) for v in values]           # whole numbers: 1.5 is no sequence
    if any(not low <= v < rows for v in values):
        raise ValueError(f"{what} must lie in [{low}, {rows}), got {values}")
    return torch.tensor(values, dtype=torch.int32, device=device)


def _move(what: str, dst: ModelCache, src: ModelCache, order, rows) -> None:
    same = dst is src
    theirs = _row_table(src)
    ours = theirs if same else _row_table(dst)
    if not same:
        if theirs not in ours.partners:
            _pair(what, ours, theirs)
        if (dst.engram_ids is None) != (src.engram_ids is None):
            raise ValueError(f"{what}: one of the caches keeps engram ids")
        ours.check(src.offset)
    visible = theirs.visible(src.offset)
    order = _index(f"{what}: order", order, theirs.batch, -1, ours.device)
    if rows is not None:
        rows = _index(f"{what}: rows", rows, ours.batch, 0, ours.device)
    elif order.numel() > ours.batch:
        raise ValueError(f"{what}: {order.numel()} rows into a cache of {ours.batch}")
    if dst.offset != src.offset and (rows is not None or order.numel() != ours.batch):
        raise ValueError(f"{what}: a cache at position {src.offset} gives single rows to one at {dst.offset}")
    engram = dst.engram_ids is not None
    if engram:
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError(f"{what}: engram ids live on the host, their order cannot be captured")
        if src.offset > dst.engram_ids.shape[1]:
            raise ValueError(f"{what}: {src.offset} positions into engram ids of {dst.engram_ids.shape[1]}")
    _abi.cache_move(theirs.pointers, ours.pointers, theirs.strides, ours.strides, visible, ours.fills, order, rows,
                    theirs.batch, ours.batch, same, ours.device)
    if engram:                             # host memory: this waits for order and rows
        o = order.cpu().numpy()
        r = np.arange(len(o)) if rows is None else rows.cpu().numpy()
        old = src.engram_ids[:, :src.offset].copy()
        for s, d in zip(o, r):
            if 0 <= d < ours.batch:
                dst.engram_ids[d, :src.offset] = old[s] if 0 <= s < theirs.batch else 0
    dst.offset = src.offset


def reorder_sequences(cache: ModelCache, order, rows=None) -> None:
    """Sequence rows[i] of the batch (row i without rows) becomes what sequence order[i] was, in every buffer of every
    layer, in place: beams that follow a survivor, a fork inside the batch, finished sequences' rows filled from the
    end. All rows are read before any is written. -1 (any order outside the batch) empties the row: its visible part is
    what a new cache holds. Rows that are not named keep theirs.

    order and rows are int32 device tensors, read by the kernel (a rows entry outside the batch then moves nothing), or
    host sequences, checked here. Of several moves to one row the last counts. Only what cache.offset positions have
    written moves; the offset stays. A captured call (device tensors) reads order and rows when it is replayed and moves
    what was visible when it was captured."""
    _move("reorder_sequences", cache, cache, order, rows)


def copy_sequences(dst: ModelCache, src: ModelCache, order, rows=None) -> None:
    """Row rows[i] of dst (row i without rows) becomes sequence order[i] of src, as reorder_sequences moves rows: a
    prompt computed once and forked into a batch, a sequence admitted into a running batch. Both caches have one
    configuration and format; batch sizes and capacities may differ. Either both are at one position, or the move names
    every row of dst (no rows, as many orders as rows) and dst takes src's position."""
    _move("copy_sequences", dst, src, order, rows)
