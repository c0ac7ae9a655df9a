"""Attention layers and the stack with their projections in 8 bits: every projection that a forward makes against the
product of its own operands in 64 bits, the stack's fused calls against the separate ones to the last bit, and the kernel
seam's 8-bit functions. (Whole outputs of two roundings are not compared: between layers the values pass the fp4 and fp8 grids
of the caches, where half a bf16 step before a border becomes a whole step of the grid, up to a third of a value.)"""

from __future__ import annotations

import pytest
import torch

from common import RELEASE_TOY, model_args

pytestmark = pytest.mark.gpu

BF = torch.bfloat16
CFG = dict(RELEASE_TOY, max_seq_len=64)
ALL = ("wq_a", "wkv", "wq_b", "wo_b")


def stack(gpu, names, layers=8):
    from dsv41.model import AttentionStack
    torch.manual_seed(5)
    s = AttentionStack(model_args(dict(CFG, n_layers=layers)), BF, gpu)
    with torch.no_grad():
        for i, layer in enumerate(s.layers):
            layer.attn_sink.normal_()
            for m in layer.modules():
                if isinstance(m, torch.nn.Linear):
                    m.weight.copy_(torch.randn(m.weight.shape, device=gpu) * m.weight.shape[1] ** -0.5)
            s.norms[i].weight.uniform_(0.5, 1.5)
    s.quantize_projections(names)
    return s


def separate(s, h, cache):
    """AttentionStack.forward from separate calls: the residual addition, the norm and the quantization one by one."""
    from dsv41 import mx8
    from dsv41.model import SharedState
    start, shared = cache.offset, SharedState()
    h = h.clone()
    for layer, norm in zip(s.layers, s.norms):
        x, _ = mx8.norm_quantize(h, norm.weight, norm.eps)
        if isinstance(layer.wo_b, mx8.MX8Linear):
            h = layer(x, start, cache, shared, residual=h)
        else:
            h = h + layer(x, start, cache, shared)
    cache.offset = start + h.shape[1]
    return h


@pytest.mark.parametrize("names", [ALL, ("wq_b",), ("wq_a", "wo_b"), ("wkv",), ("wq_a", "wkv")])
def test_stack_with_8_bit_projections(gpu, names):
    """Prompt, a second chunk and single tokens through the released topology at toy size."""
    s = stack(gpu, names)
    g = torch.Generator(device=gpu).manual_seed(6)
    c0, c1 = s.make_cache(3), s.make_cache(3)
    for n in (13, 6, 1, 1, 1):
        h = torch.randn(3, n, CFG["dim"], generator=g, device=gpu).to(BF)
        before = h.clone()
        y = s(h, c0)
        assert torch.equal(h, before)            # the caller's rows stay
        assert y.isfinite().all() and torch.equal(y, separate(s, h, c1)), (names, n)


def test_every_projection_multiplies_its_own_rows(gpu):
    """Hooks on the 8-bit projections see what each was given: its output is the product of that (2^-8 of the result: half a
    bf16 step; 7 * 2^-13 of sum |x w|: each of eight neighbouring products but the largest may lose 2^-13 of that one),
    wq_b's rows are the norm of wq_a's."""
    from dsv41 import mx8
    s = stack(gpu, ALL)
    seen = {}

    def hook(name):
        def see(lin, args, kwargs, out):
            q = args[0] if isinstance(args[0], mx8.Quantized) else mx8.quantize(args[0])
            r = kwargs.get("residual")
            seen.setdefault(name, []).append((lin, q, out.clone(), None if r is None else before.pop()))
        return see

    before = []
    for i, layer in enumerate(s.layers):
        for name in ALL:
            getattr(layer, name).register_forward_hook(hook((i, name)), with_kwargs=True)
        layer.wo_b.register_forward_pre_hook(lambda lin, args, kwargs: before.append(kwargs["residual"].clone()),
                                             with_kwargs=True)
    cache = s.make_cache(2)
    g = torch.Generator(device=gpu).manual_seed(6)
    for n in (13, 1):
        s(torch.randn(2, n, CFG["dim"], generator=g, device=gpu).to(BF), cache)
    assert len(seen) == 8 * 4 and all(len(v) == 2 for v in seen.values())
    for (i, name), calls in seen.items():
        for at, (lin, q, out, residual) in enumerate(calls):
            x = mx8.dequantize(q, torch.float32).double()
            w = lin.weight_values(torch.float32).double()
            want, size = x @ w.t(), x.abs() @ w.abs().t()
            if name == "wo_b":
                want = want + residual.double()
            assert ((out.double() - want).abs() <= 2.0 ** -8 * want.abs() + 7 * 2.0 ** -13 * (1 + 2.0 ** -8) * size).all()
            if name == "wq_b":
                layer = s.layers[i]
                rows = layer.q_norm(seen[i, "wq_a"][at][2])
                assert all(torch.equal(a, b) for a, b in zip(q, mx8.quantize(rows)))
            if name == "wkv":
                assert all(torch.equal(a, b) for a, b in zip(q, seen[i, "wq_a"][at][1]))


def test_layer_takes_rows_in_8_bits_and_a_residual(gpu):
    """The rows in 8 bits, given or made inside, are the same call; the residual added inside wo_b's launch is the output
    added to it, rounded once (half a step of the sum from the separate addition's two roundings)."""
    from dsv41 import mx8
    from dsv41.model import SharedState
    got = stack(gpu, ALL, 1)
    layer = got.layers[0]
    g = torch.Generator(device=gpu).manual_seed(7)
    x = torch.randn(2, 5, CFG["dim"], generator=g, device=gpu).to(BF)
    r = torch.randn(2, 5, CFG["dim"], generator=g, device=gpu).to(BF)

    def call(**kw):
        return layer(x, 0, got.make_cache(2), SharedState(), **kw)

    y = call()
    assert layer.takes_quantized and torch.equal(call(x8=mx8.quantize(x)), y)
    held = r.clone()
    out = call(residual=held)
    assert out is held
    want = y.double() + r.double()
    assert ((out.double() - want).abs() <= 2.0 ** -8 * (want.abs() + y.double().abs())).all()


def test_stack_with_8_bit_projections_in_a_graph(gpu):
    """One-token steps captured and replayed, with eager steps between: every replay equals the eager step."""
    from dsv41.cache import restore, snapshot
    got = stack(gpu, ALL, 2)
    g = torch.Generator(device=gpu).manual_seed(8)
    cache = got.make_cache(2)
    got(torch.randn(2, 9, CFG["dim"], generator=g, device=gpu).to(BF), cache)
    h = torch.randn(2, 1, CFG["dim"], generator=g, device=gpu).to(BF)
    held = snapshot(cache)
    got(h, cache)
    restore(cache, held)
    torch.cuda.synchronize()
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph, stream=side):
        y = got(h, cache)
    for i in range(3):
        h.copy_(torch.randn(2, 1, CFG["dim"], generator=g, device=gpu).to(BF))
        restore(cache, held)
        want = got(h, cache).clone()
        restore(cache, held)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want)


def test_adapters_and_8_bit_projections_keep_apart(gpu):
    got = stack(gpu, ("wq_b",), 1)
    with pytest.raises(ValueError, match="8 bits"):
        got.add_adapters(2, 8)
    got.add_adapters(2, 8, ("wq_a", "wo_b"))
    with pytest.raises(ValueError, match="adapters"):
        got.quantize_projections(("wo_b",))
    h = torch.randn(2, 4, CFG["dim"], device=gpu).to(BF)
    got(h, got.make_cache(2), torch.tensor([0, -1], dtype=torch.int32, device=gpu))


def test_kernel_seam_in_8_bits(gpu):
    """act_quant's codes and scales and fp8_gemm, in torch's own types, as the reference model's linear calls them."""
    import dsv41.kernel as K
    from dsv41 import mx8
    g = torch.Generator(device=gpu).manual_seed(9)
    x = torch.randn(3, 7, 160, generator=g, device=gpu).to(BF)
    w = mx8.quantize_weight((torch.randn(72, 160, generator=g, device=gpu) * 0.1).to(BF))
    codes, scales = K.act_quant(x, 32, "ue8m0", torch.float8_e8m0fnu)
    assert codes.dtype == torch.float8_e4m3fn and scales.dtype == torch.float8_e8m0fnu and scales.shape == (3, 7, 5)
    values = codes.double() * scales.double().repeat_interleave(32, -1)
    assert torch.equal(values.to(BF), K.act_quant(x.clone(), 32, "ue8m0", None, True))
    y = K.fp8_gemm(codes, scales, w.codes.view(torch.float8_e4m3fn), w.scales.view(torch.float8_e8m0fnu))
    assert torch.equal(y, mx8.MX8Linear(*w)(x)) and y.dtype == BF
    wv = mx8.dequantize(w, torch.float32).double()
    want = values @ wv.t()
    assert ((y.double() - want).abs() <= 2.0 ** -8 * want.abs() + 7 * 2.0 ** -13 * (values.abs() @ wv.abs().t())).all()
    with pytest.raises(NotImplementedError):
        K.act_quant(x, 128, "ue8m0")
    with pytest.raises(NotImplementedError):
        K.fp8_gemm(codes, scales.float(), codes[0], scales[0].float())
