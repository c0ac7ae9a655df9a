"""Performance cases of what a serving program does for a batch of unlike requests: each sequence under its own
low-rank adapter, and sequences that are forked, admitted, moved and freed in the caches.

A case is a dict of plain values; ``op`` says which operator it goes through:

* ``linear``   ``adapter_linear``: one projection of the attention layer with one adapter (or none) per sequence;
* ``pair``     ``adapter_linear_pair``: ``wq_a`` and ``wkv`` on the same rows, each with its own bank of adapters;
* ``reorder``  ``reorder_sequences``: the rows of one cache moved in place (beams, compaction), rows emptied;
* ``copy``     ``copy_sequences``: rows of one cache into another (a prompt forked, a sequence admitted).

Widths are the released configuration's (hidden 5120, q rank 1280, 64 heads of 512, output rank 8 x 1024) and the tiny
float32 configuration's (hidden 256); caches are the 40-layer stack's (four owners, ratio 4) and a 4-layer one's.
"""

from __future__ import annotations

import math
import os
import sys

import torch

own = False

BF, F32, U8 = torch.bfloat16, torch.float32, torch.uint8
SHAPES = {"wq_a": (5120, 1280), "wkv": (5120, 512), "wq_b": (1280, 32768), "wo_b": (8192, 5120),
          "tiny_wq": (256, 128), "tiny_wo": (64, 256)}
WIN, DI, RATIO = 128, 128, 4


def _package():
    """The framework's modules; its folder is not on the path by itself."""
    root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "deepseek-v41-mlx_amd")
    if root not in sys.path:
        sys.path.insert(0, root)
    from dsv41 import adapters, cache, config
    return adapters, cache, config


# ---------------------------------------------------------------------------- the cases


def listed():
    return [
        # one user's token through wq_a and wkv under one adapter: the smallest serving call, launches and latency
        dict(name="pair_b1_r16", op="pair", proj="wq_a", batch=1, n=1, slots=4, rank=16, none=0),
        # a ragged batch of short decode calls, two sequences without an adapter
        dict(name="pair_b17_r8", op="pair", proj="wq_a", batch=17, n=1, slots=8, rank=8, none=2),
        # a full decode batch, every sequence another adapter, on the widest projection
        dict(name="wq_b_b64_r16", op="linear", proj="wq_b", batch=64, n=1, slots=64, rank=16, none=0),
        # an odd batch under few large adapters on the output projection
        dict(name="wo_b_b33_r64", op="linear", proj="wo_b", batch=33, n=1, slots=8, rank=64, none=5),
        # one prompt under one adapter
        dict(name="wq_a_prompt_4k_r16", op="linear", proj="wq_a", batch=1, n=4096, slots=4, rank=16, none=0),
        # three short prompts of an odd length, tiles that hold two of them, one without an adapter
        dict(name="wq_b_3x333_r32", op="linear", proj="wq_b", batch=3, n=333, slots=8, rank=32, none=1),
        # two long prompts under large adapters: the largest call
        dict(name="wo_b_8k_r64", op="linear", proj="wo_b", batch=2, n=4096, slots=4, rank=64, none=0),
        # the tiny float32 configuration's prompt
        dict(name="tiny_f32_b2", op="linear", proj="tiny_wq", batch=2, n=128, slots=4, rank=4, none=0),
        # a beam search step early in a chat: 4 beams, 500 tokens, all 40 layers
        dict(name="beams_b4_500", op="reorder", batch=4, ctx=500, layers=40, fmt="dense", how="beams"),
        # finished sequences leave a full batch: rows from the end fill the holes, the rest are emptied
        dict(name="compact_b64_64k_packed", op="reorder", batch=64, ctx=65536, layers=40, fmt="packed", how="compact"),
        # a prompt computed once and forked into 16 continuations
        dict(name="fork_b16_16k", op="copy", batch=16, ctx=16384, layers=40, fmt="dense", how="fork"),
        # one long sequence admitted into a running batch over the fp8 cache
        dict(name="admit_b16_128k_fp8", op="copy", batch=16, ctx=131071, layers=40, fmt="fp8", how="admit"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("linear", "linear", "pair", "reorder", "copy"))
    if op in ("linear", "pair"):
        proj = "wq_a" if op == "pair" else rng.choice(("wq_a", "wkv", "wq_b", "wo_b", "tiny_wq", "tiny_wo"))
        if rng.random() < 0.5:
            batch, n = _log(rng, 1, 128), 1
        else:
            batch = rng.choice((1, 1, 2, 3, 7))
            n = _log(rng, 2, 8192 // batch if proj != "wq_b" else 4096 // batch)
        return dict(op=op, proj=proj, batch=batch, n=n, slots=_log(rng, 1, 64), rank=rng.choice((4, 8, 12, 16, 32, 64)),
                    none=rng.choice((0, 0, batch // 4)))
    fmt, layers = rng.choice(("dense", "fp8", "packed")), rng.choice((4, 40))
    how = rng.choice(("beams", "compact")) if op == "reorder" else rng.choice(("fork", "admit"))
    while True:
        c = dict(op=op, batch=_log(rng, 2, 64), ctx=_log(rng, 1, 131072), layers=layers, fmt=fmt, how=how)
        if c["batch"] * sum(_row_bytes(c)) <= 1 << 31:
            return c


# ---------------------------------------------------------------------------- adapters


def _ids(c, g):
    """One adapter per sequence, as many different ones as there are, -1 for ``none`` of the sequences."""
    b = c["batch"]
    ids = (torch.arange(b, dtype=torch.int32) % c["slots"])
    ids[:c["none"]] = -1
    return ids[torch.randperm(b, generator=g)].contiguous()


def _projections(c):
    return ("wq_a", "wkv") if c["op"] == "pair" else (c["proj"],)


def _adapter_inputs(c, seed):
    cpu = torch.Generator().manual_seed(seed)
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = F32 if c["proj"].startswith("tiny") else BF

    def normal(*shape, scale=1.0):
        return torch.randn(*shape, generator=g, device="cuda").mul_(scale).to(dt)

    ids = _ids(c, cpu).cuda()
    k = SHAPES[c["proj"]][0]
    s = dict(ids=ids, x=normal(c["batch"], c["n"], k), w=[], a=[], b=[], scale=[])
    for p in _projections(c):
        n = SHAPES[p][1]
        s["w"].append(normal(n, k, scale=0.02))
        s["a"].append(normal(c["slots"], c["rank"], k, scale=0.02))
        s["b"].append(normal(c["slots"], n, c["rank"], scale=0.02))
        s["scale"].append(0.5 + 2.0 * torch.rand(c["slots"], generator=g, device="cuda"))
    return s


def _adapted(x, w, a, b, scale, ids):
    """x w^T + scale (x A^T) B^T with the sequence's own A and B, in 32 bits, rounded once."""
    dt, slot = x.dtype, ids.clamp(min=0).long()
    x = x.float()
    h = torch.matmul(x, a[slot].float().transpose(1, 2))
    delta = torch.matmul(h, b[slot].float().transpose(1, 2)) * scale[slot][:, None, None]
    return (torch.matmul(x, w.float().t()) + torch.where(ids[:, None, None] >= 0, delta, 0.0)).to(dt)


# ---------------------------------------------------------------------------- caches


def _topology(c):
    """Layers, their compress ratios, the owners, the KV width."""
    if c["layers"] == 40:
        return (0, 0) + (RATIO,) * 38, (2, 8, 14, 20), 512
    return (RATIO,) * 4, (0,), 64


def _buffers(c):
    """(layer, name, rows per sequence, visible rows, bytes or values per row, type) of every cache buffer."""
    ratios, owners, d = _topology(c)
    cap, ctx = c["ctx"] + 64, c["ctx"]
    nc, vc, wp = cap // RATIO, ctx // RATIO, min(ctx, WIN)
    dense, fp8, packed = (c["fmt"] == f for f in ("dense", "fp8", "packed"))
    found = []
    for l in range(len(ratios)):
        found.append((l, "win_kv8", WIN, wp, d + d // 32, U8) if packed else (l, "win_kv", WIN, wp, d, BF))
        if l in owners:
            if dense:
                found += [(l, "comp_kv", nc, vc, d, BF), (l, "index_k", nc, vc, DI, BF)]
            if fp8:
                found += [(l, "comp_kv8", nc, vc, d, U8), (l, "comp_ks", -(-nc // 32), -(-vc // 32), d // 32, U8),
                          (l, "index_k8", nc, vc, DI, U8), (l, "index_k8s", -(-nc // 32), -(-vc // 32), DI // 32, U8)]
            if packed:
                found += [(l, "comp_kv4", nc, vc, d // 2 + d // 16, U8), (l, "index_k4", nc, vc, DI // 2, U8),
                          (l, "index_ks", nc, vc, DI // 32, U8)]
            found += [(l, "kv_state", RATIO, RATIO, d, F32), (l, "score_state", RATIO, RATIO, d, F32)]
    return found


def _row_bytes(c):
    """Visible bytes of one sequence, buffer by buffer."""
    return [v * w * t.itemsize for _, _, _, v, w, t in _buffers(c)]


def _moves(c, g):
    """(order, rows): row rows[i] of the destination takes row order[i] of the source, or is emptied (-1). Rows that are
    read keep their place, as a scheduler that moves as little as it can leaves them."""
    b = c["batch"]
    if c["how"] == "fork":
        return [0] * b, list(range(b))
    if c["how"] == "admit":
        return [0], [int(torch.randint(0, b, (1,), generator=g))]
    if c["how"] == "beams":                # groups of up to 4 beams; the survivors stay, the others take a survivor
        order = []
        for at in range(0, b, 4):
            m = min(4, b - at)
            alive = torch.randperm(m, generator=g)[:max(1, m // 2)].tolist()
            order += [at + (i if i in alive else alive[i % len(alive)]) for i in range(m)]
        return order, list(range(b))
    keep = sorted(torch.randperm(b, generator=g)[:max(1, 5 * b // 8)].tolist())
    holes = [i for i in range(len(keep)) if i not in keep]
    late = [i for i in keep if i >= len(keep)]
    dead = [i for i in range(len(keep), b) if i not in keep]
    return late + [-1] * len(dead), holes + dead


def _cache_tensors(c, batch, g):
    return [torch.randint(0, 256, (batch, n, w), generator=g, device="cuda", dtype=U8) if t == U8 else
            torch.randn(batch, n, w, generator=g, device="cuda", dtype=t) for _, _, n, _, w, t in _buffers(c)]


def _source_batch(c):
    return 1 if c["op"] == "copy" else c["batch"]


def _cache_inputs(c, seed):
    cpu = torch.Generator().manual_seed(seed)
    g = torch.Generator(device="cuda").manual_seed(seed)
    order, rows = _moves(c, cpu)
    s = dict(order=torch.tensor(order, dtype=torch.int32, device="cuda"),
             rows=torch.tensor(rows, dtype=torch.int32, device="cuda"))
    s["dst"] = _cache_tensors(c, c["batch"], g)
    s["src"] = _cache_tensors(c, 1, g) if c["op"] == "copy" else s["dst"]
    return s


def _model_cache(c, batch, tensors):
    """A ModelCache that holds these tensors."""
    _, cache, config = _package()
    ratios, owners, d = _topology(c)
    args = config.ModelArgs(n_layers=len(ratios), head_dim=d, window_size=WIN, compress_ratios=ratios,
                            kv_source_layers=owners, index_source_layers=owners, index_head_dim=DI, engram_layer_ids=())
    m = cache.ModelCache(args, batch, c["ctx"] + 64, BF, "cuda", "mxfp4" if c["fmt"] == "packed" else "dense", c["fmt"],
                         32 if c["fmt"] == "fp8" else 1)
    for (l, name, *_), t in zip(_buffers(c), tensors):
        setattr(m.layers[l].comp_state if name.endswith("_state") else m.layers[l], name, t)
    m.offset = c["ctx"]
    return m


def _moved(name, dst, src, visible, order, rows):
    """One buffer's rows, all read before any is written; the emptied ones as a new cache holds them."""
    got = src[order.clamp(min=0).long(), :visible]
    got = torch.where(order[:, None, None] >= 0, got, torch.full_like(got, -math.inf if name == "score_state" else 0))
    dst[rows.long(), :visible] = got
    return dst


# ---------------------------------------------------------------------------- the interface


def prepare(case, seed):
    c = case
    if c["op"] in ("linear", "pair"):
        s = _adapter_inputs(c, seed)
        if own:
            adapters = _package()[0]
            s["lin"], s["bank"] = [], []
            for w, a, b, scale in zip(s["w"], s["a"], s["b"], s["scale"]):
                lin = torch.nn.Linear(1, 1, bias=False)
                lin.weight = torch.nn.Parameter(w, requires_grad=False)
                bank = adapters.AdapterBank(c["slots"], w.shape[1], w.shape[0], c["rank"], w.dtype, "cuda")
                for t in range(c["slots"]):
                    bank.load(t, a[t], b[t], float(scale[t]))
                s["lin"].append(lin)
                s["bank"].append(bank)
    else:
        s = _cache_inputs(c, seed)
        if own:
            s["dst_cache"] = _model_cache(c, c["batch"], s["dst"])
            s["src_cache"] = _model_cache(c, 1, s["src"]) if c["op"] == "copy" else s["dst_cache"]
    s["case"] = c
    return s


def run(state):
    s, c = state, state["case"]
    if own:
        adapters, cache, _ = _package()
        if c["op"] == "linear":
            return adapters.adapter_linear(s["lin"][0], s["x"], s["bank"][0], s["ids"])
        if c["op"] == "pair":
            return adapters.adapter_linear_pair(s["lin"][0], s["lin"][1], s["x"], s["bank"][0], s["bank"][1], s["ids"])
        if c["op"] == "reorder":
            cache.reorder_sequences(s["dst_cache"], s["order"], s["rows"])
        else:
            cache.copy_sequences(s["dst_cache"], s["src_cache"], s["order"], s["rows"])
        return s["dst"]
    if c["op"] in ("linear", "pair"):
        y = tuple(_adapted(s["x"], w, a, b, scale, s["ids"])
                  for w, a, b, scale in zip(s["w"], s["a"], s["b"], s["scale"]))
        return y if c["op"] == "pair" else y[0]
    return [_moved(name, d, t, v, s["order"], s["rows"])
            for (_, name, _, v, _, _), d, t in zip(_buffers(c), s["dst"], s["src"])]


def work(case):
    c = case
    if c["op"] in ("linear", "pair"):
        rows, size = c["batch"] * c["n"], 4 if c["proj"].startswith("tiny") else 2
        live = c["batch"] - c["none"]
        distinct, r = min(live, c["slots"]), c["rank"]
        k = SHAPES[c["proj"]][0]
        values, flops = rows * k, 0
        for p in _projections(c):
            n = SHAPES[p][1]
            values += n * k + rows * n + distinct * r * (k + n)
            flops += 2 * rows * k * n + 2 * live * c["n"] * r * (k + n)
        return {"bytes": size * values + 4 * c["batch"], "flops": flops}
    order, rows = _moves(c, torch.Generator().manual_seed(0))
    read = len({o for o, r in zip(order, rows) if o >= 0 and (c["op"] == "copy" or o != r)})
    written = sum(1 for o, r in zip(order, rows) if c["op"] == "copy" or o != r)
    return {"bytes": (read + written) * sum(_row_bytes(c)), "flops": 0}


def exact(case, seed):
    c = case
    if c["op"] in ("linear", "pair"):
        s = _adapter_inputs(c, seed)
        found = []
        for w, a, b, scale in zip(s["w"], s["a"], s["b"], s["scale"]):
            y = s["x"].double() @ w.double().t()
            for i, t in enumerate(s["ids"].tolist()):
                if t >= 0:
                    y[i] += float(scale[t]) * ((s["x"][i].double() @ a[t].double().t()) @ b[t].double().t())
            found.append(y)
        return tuple(found) if c["op"] == "pair" else found[0]
    s = _cache_inputs(c, seed)
    found = []
    for (_, name, _, v, _, _), d, t in zip(_buffers(c), s["dst"], s["src"]):
        new = d.clone()
        for o, r in zip(s["order"].tolist(), s["rows"].tolist()):
            if o >= 0:
                new[r, :v] = t[o, :v]
            else:
                new[r, :v] = -math.inf if name == "score_state" else 0
        found.append(new)
    return found
