"""Low-rank adapters of many sequences beside the shared projections (wq_a, wkv, wq_b and wo_b of
attention.py:114-122 and :179).

A bank holds the adapters of one projection, one per slot; a call gives every sequence of the batch its own slot, or
none:

    y = x w^T + scale[t] (x A[t]^T) B[t]^T,   t = ids[sequence], t outside the slots: y = x w^T

``ids`` is an int32 device tensor, read by the kernels, so a captured HIP graph replays with whatever it then holds.
The rank-wide product and all sums are float32; the result is rounded once where the projection itself runs here, and
once more where it is torch's (float32 activations, widths the matrix-core kernels do not take, a module with hooks).
Inference only: a call that autograd would have to follow - x, the projection or a bank requires gradients or holds a
tangent - is refused.
"""

from __future__ import annotations

import torch

from . import _abi
from .layers import decode_linear, decode_linear_pair


class AdapterBank:
    """The adapters of one projection: ``a`` [slots, rank, in], ``b`` [slots, out, rank], ``scale`` [slots] float32,
    all zero (a slot that changes nothing) until loaded. Ranks are stored in multiples of 8, zero padded."""

    def __init__(self, slots: int, in_features: int, out_features: int, rank: int, dtype=torch.bfloat16,
                 device="cuda"):
        if slots < 1 or in_features < 1 or out_features < 1 or rank < 1:
            raise ValueError(f"AdapterBank: slots {slots}, in {in_features}, out {out_features} and rank {rank} must be "
                             "positive")
        if dtype not in (torch.bfloat16, torch.float32):
            raise ValueError(f"AdapterBank: dtype {dtype} not supported (float32 or bfloat16)")
        self.slots, self.in_features, self.out_features, self.rank = slots, in_features, out_features, rank
        held = -(-rank // 8) * 8
        self.a = torch.zeros(slots, held, in_features, dtype=dtype, device=device)
        self.b = torch.zeros(slots, out_features, held, dtype=dtype, device=device)
        self.scale = torch.zeros(slots, dtype=torch.float32, device=device)

    def _slot(self, slot: int) -> int:
        if not 0 <= slot < self.slots:
            raise ValueError(f"AdapterBank: slot {slot} of {self.slots}")
        return slot

    @torch.no_grad()
    def load(self, slot: int, a: torch.Tensor, b: torch.Tensor, scale: float = 1.0) -> None:
        """Puts the adapter a [r, in], b [out, r] (r at most the bank's rank) into a slot."""
        slot = self._slot(slot)
        if (a.dim() != 2 or b.dim() != 2 or a.shape[0] != b.shape[1] or a.shape[1] != self.in_features
                or b.shape[0] != self.out_features or a.shape[0] > self.rank):
            raise ValueError(f"AdapterBank: a {tuple(a.shape)} and b {tuple(b.shape)} are no adapter of rank at most "
                             f"{self.rank} of [{self.out_features}, {self.in_features}]")
        r = a.shape[0]
        self.a[slot, :r].copy_(a)
        self.a[slot, r:].zero_()
        self.b[slot, :, :r].copy_(b)
        self.b[slot, :, r:].zero_()
        self.scale[slot] = scale

    @torch.no_grad()
    def clear(self, slot: int) -> None:
        """Empties a slot: sequences under it get the plain projection."""
        slot = self._slot(slot)
        self.a[slot].zero_()
        self.b[slot].zero_()
        self.scale[slot] = 0.0


_forward_ad = torch.autograd.forward_ad


def _no_gradient(x: torch.Tensor, w: torch.Tensor, bank: AdapterBank | None = None) -> None:
    """Refuses operands of a call that autograd would have to follow, backward or forward."""
    if torch.is_grad_enabled() and (x.requires_grad or w.requires_grad or bank is not None and (
            bank.a.requires_grad or bank.b.requires_grad or bank.scale.requires_grad)):
        raise ValueError("adapter projections are not differentiable: call them under torch.no_grad()")
    if _forward_ad._current_level >= 0:
        held = (x, w) if bank is None else (x, w, bank.a, bank.b, bank.scale)
        if any(_forward_ad.unpack_dual(t).tangent is not None for t in held):
            raise ValueError("adapter projections are not differentiable: their operands may hold no tangent")


_module = torch.nn.modules.module
_FORWARD_HOOKS = ("_forward_hooks", "_forward_pre_hooks", "_backward_hooks", "_backward_pre_hooks")


# multiply-adds up to which a product off the bf16 tiles' shapes runs with its adapters in one launch
# (dsv41_adapter_plain) instead of after torch's linear
_PLAIN_MACS = 1 << 28


def _product_weight(lin: torch.nn.Linear, x: torch.Tensor) -> torch.Tensor | None:
    """The projection's weight where the module's call is the product alone (no hooks, bias or forward of its own), of
    x's type and in one piece, so that a kernel may stand in for the module."""
    own = lin.__dict__
    params = own["_parameters"]            # a weight or bias that is no parameter (a plain tensor in its place) is not there
    w = params.get("weight")
    if (type(lin) is not torch.nn.Linear or "forward" in own or any(own[h] for h in _FORWARD_HOOKS)
            or _module._global_forward_hooks or _module._global_forward_pre_hooks or params.get("bias", own) is not None):
        return None
    return w if w is not None and w.dtype is x.dtype and w.is_contiguous() else None


def _tiles_ok(w: torch.Tensor, x: torch.Tensor, rank: int) -> bool:
    """What dsv41_adapter_linear takes: bf16 in whole 64-channel steps and 32-row weight tiles, 16-byte addresses."""
    n, k = w.shape
    return (x.dtype is torch.bfloat16 and rank <= 128 and k % 64 == 0 and n % 32 == 0 and w.data_ptr() % 16 == 0
            and x.data_ptr() % 16 == 0)


def adapter_linear(lin: torch.nn.Linear, x: torch.Tensor, bank: AdapterBank | None, ids: torch.Tensor | None,
                   wide_only: bool = False) -> torch.Tensor:
    """lin(x) with every sequence's own adapter: x [sequences, (tokens,) in], ids int32 [sequences]. Without a bank or
    ids it is decode_linear(lin, x, wide_only)."""
    if bank is None or ids is None:
        return decode_linear(lin, x, wide_only)
    x = x.contiguous()
    w = _product_weight(lin, x)
    if w is not None:
        _no_gradient(x, w, bank)
        if _tiles_ok(w, x, bank.a.shape[1]):
            return _abi.adapter_linear(x, w, bank.a, bank.b, bank.scale, ids)
        if x.numel() * w.shape[0] <= _PLAIN_MACS:
            return _abi.adapter_plain(x, w, bank.a, bank.b, bank.scale, ids)
    _no_gradient(x, lin.weight, bank)
    if (bank.out_features, bank.in_features) != tuple(lin.weight.shape):
        raise ValueError(f"adapters of [{bank.out_features}, {bank.in_features}] on a projection of "
                         f"{list(lin.weight.shape)}")
    y = lin(x).contiguous()
    _no_gradient(y, lin.weight)                # a bias, or what a module of its own multiplies with
    return _abi.adapter_add(x, bank.a, bank.b, bank.scale, ids, y)


def adapter_linear_pair(lin0: torch.nn.Linear, lin1: torch.nn.Linear, x: torch.Tensor, bank0: AdapterBank | None,
                        bank1: AdapterBank | None, ids: torch.Tensor | None):
    """(adapter_linear(lin0, x, bank0, ids), adapter_linear(lin1, x, bank1, ids)) in one call where both run on the bf16
    tiles; without any bank or ids it is decode_linear_pair."""
    if ids is None or (bank0 is None and bank1 is None):
        return decode_linear_pair(lin0, lin1, x)
    x = x.contiguous()
    w0, w1 = _product_weight(lin0, x), _product_weight(lin1, x)
    if (w0 is not None and w1 is not None and w0.shape[1] == w1.shape[1]
            and _tiles_ok(w0, x, 0 if bank0 is None else bank0.a.shape[1])
            and _tiles_ok(w1, x, 0 if bank1 is None else bank1.a.shape[1])):
        _no_gradient(x, w0, bank0)
        _no_gradient(x, w1, bank1)
        return _abi.adapter_linear_pair(x, w0, w1, None if bank0 is None else (bank0.a, bank0.b, bank0.scale),
                                        None if bank1 is None else (bank1.a, bank1.b, bank1.scale), ids)
    return adapter_linear(lin0, x, bank0, ids), adapter_linear(lin1, x, bank1, ids)
