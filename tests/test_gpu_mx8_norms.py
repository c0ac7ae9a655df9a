"""Norms with hooks, or of a formula of their own, beside 8-bit projections: the modules are called, as without 8 bits, and what
they give is what is quantized."""

from __future__ import annotations

import pytest
import torch

from test_gpu_mx8_layers import ALL, BF, CFG, stack

pytestmark = pytest.mark.gpu


def called(s, h, cache):
    """AttentionStack.forward with every norm called and its rows handed on as they are."""
    from dsv41.model import SharedState
    start, shared = cache.offset, SharedState()
    h = h.clone()
    for layer, norm in zip(s.layers, s.norms):
        y = layer(norm(h), start, cache, shared)
        h = h + y
    cache.offset = start + h.shape[1]
    return h


def rows(n, seed):
    return torch.randn(2, n, CFG["dim"], generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda").to(BF)


@pytest.mark.parametrize("names", [ALL, ("wq_b",), ("wq_a", "wkv"), ()])
def test_hooks_of_norms_run(gpu, names):
    s = stack(gpu, names)
    seen = []
    for i, layer in enumerate(s.layers):
        for what, norm in ((("norm", i), s.norms[i]), (("q_norm", i), layer.q_norm)):
            norm.register_forward_hook(lambda m, args, out, what=what: seen.append((what, args[0].clone(), out.clone())))
    cache = s.make_cache(2)
    for n in (13, 1):
        seen.clear()
        s(rows(n, 6), cache)
        assert [w for w, *_ in seen] == [(w, i) for i in range(len(s.layers)) for w in ("norm", "q_norm")]
        for (what, i), x, y in seen:
            norm = s.norms[i] if what == "norm" else s.layers[i].q_norm
            v = x.double()
            want = norm.weight.double() * v / (v.square().mean(-1, keepdim=True) + norm.eps).sqrt()
            assert ((y.double() - want).abs() <= 2.0 ** -7 * want.abs()).all()


def test_a_norm_of_another_formula_is_called(gpu):
    """Rows twice as large, in every norm: through a subclass, a forward of its own and a hook that changes the output. The
    projections see them: the same as without 8 bits around them."""
    from dsv41.layers import RMSNorm

    class Twice(RMSNorm):
        def forward(self, x):
            return super().forward(x) * 2

    def by_class(m):
        m.__class__ = Twice

    def by_forward(m):
        m.forward = lambda x: RMSNorm.forward(m, x) * 2

    def by_hook(m):
        m.register_forward_hook(lambda _, args, y: y * 2)

    outs = []
    for change in (by_class, by_forward, by_hook, None):
        s = stack(gpu, ("wq_a", "wkv", "wq_b"))
        if change is not None:
            for m in [*s.norms, *(layer.q_norm for layer in s.layers)]:
                change(m)
        c0, c1 = s.make_cache(2), s.make_cache(2)
        for n in (13, 1):
            y = s(rows(n, 7), c0)
            if change is not None:
                assert torch.equal(y, called(s, rows(n, 7), c1))
        outs.append(y)
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2]) and not torch.equal(outs[0], outs[3])


def test_hooks_leave_the_results(gpu):
    """Without 8 bits a hooked norm's rows are the fused launch's, bit for bit."""
    plain, hooked = stack(gpu, ()), stack(gpu, ())
    for m in hooked.norms:
        m.register_forward_hook(lambda m, args, y: None)
    c0, c1 = plain.make_cache(2), hooked.make_cache(2)
    for n in (13, 1):
        assert torch.equal(plain(rows(n, 8), c0), hooked(rows(n, 8), c1))
