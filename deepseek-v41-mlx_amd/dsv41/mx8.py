"""Projections in 8 bits, in the form the release stores its weights and multiplies them (quant_method fp8, weight blocks of
32 x 32, ue8m0 scales, activations quantized as they come; docs/reference/model.py's linear over kernel.py:40-124 and
:207-307).

A tensor in 8 bits is a ``Quantized``: e4m3 codes and power-of-two scale bytes, both uint8,

    value = e4m3(code) * 2^(scale - 127)

with one scale per 32 channels of a row (activations), or per 32 x 32 block (weights). A block's scale is the smallest power of
two for which its largest value is at most 448; a block that holds an infinity or NaN reads back as NaN.

* ``quantize`` (rows), ``quantize_weight`` and ``dequantize`` convert;
* ``norm_quantize`` ends a residual addition and RMS norm in 8 bits;
* ``MX8Linear`` multiplies 8-bit rows with an 8-bit weight on the block-scaled matrix instructions, in bf16 out, with bias,
  activation and residual in the same launch; ``linear_pair`` two of them on the same rows.

Float rows may be float32 or bf16. Everything is inference only. Products accumulate in float32 over the matrix instruction's
own sums, which cut off of eight neighbouring products what lies under 2^-13 of the largest (1.4e-5 of a result on normal
values, 7 * 2^-13 of sum |x w| at worst); outputs are bf16, rounded once.
"""

from __future__ import annotations

import typing

import torch

from . import _abi

_forward_ad = torch.autograd.forward_ad


class Quantized(typing.NamedTuple):
    """codes [..., k] and scales [..., k/32] (rows) or [ceil(n/32), k/32] (a weight [n, k]), uint8."""

    codes: torch.Tensor
    scales: torch.Tensor


def _no_gradient(*tensors) -> None:
    """Refuses operands of a call that autograd would have to follow, backward or forward."""
    for t in tensors:
        if t is None:
            continue
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"8-bit projections take tensors, got {type(t).__name__}")
        if t.requires_grad and torch.is_grad_enabled():
            raise ValueError("8-bit projections are not differentiable: call them under torch.no_grad()")
    if _forward_ad._current_level >= 0 and any(t is not None and _forward_ad.unpack_dual(t).tangent is not None
                                               for t in tensors):
        raise ValueError("8-bit projections are not differentiable: their operands may hold no tangent")


def quantize(x: torch.Tensor) -> Quantized:
    """Rows x [..., k] in 8 bits, one scale per 32 channels (act_quant without inplace)."""
    _no_gradient(x)
    return Quantized(*_abi.quant_mx8(x.contiguous()))


def quantize_weight(w: torch.Tensor) -> Quantized:
    """A weight w [n, k] in 8 bits, one scale per 32 x 32 block."""
    _no_gradient(w)
    return Quantized(*_abi.quant_mx8_blocks(w.contiguous()))


def dequantize(q: Quantized, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The values of rows or of a weight in 8 bits (exact in both types, but for bf16 magnitudes under 2^-126)."""
    return _abi.dequant_mx8(q[0], q[1], dtype)


def norm_quantize(x: torch.Tensor, weight: torch.Tensor, eps: float, delta: torch.Tensor | None = None,
                  rows: bool = True):
    """(y, Quantized): y = the RMS norm of the rows x [..., dim], or with delta of the residual addition, x <- x + delta in
    place, and quantize(y). Rows are the formula's, rounded to x's type: a border between two codes is no place for a float32
    sum's error (RMSNorm's rows may be a step of that type off). eps counts as float32. Without rows, y is not written and None."""
    _no_gradient(x, weight, delta)
    y, codes, scales = _abi.rmsnorm_mx8(x, weight, eps, delta, rows)
    return y, Quantized(codes, scales)


class MX8Linear(torch.nn.Module):
    """A projection whose weight [n, k] is held in 8 bits: codes [n, k] and scales [ceil(n/32), k/32] (or [n, k/32]) as the
    release's checkpoint has them (viewed as uint8), and a float32 bias or none. The tensors are kept, not copied."""

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, bias: torch.Tensor | None = None):
        super().__init__()
        name = "MX8Linear"
        if codes.dtype != torch.uint8 or scales.dtype != torch.uint8:
            raise ValueError(f"{name}: codes and scales must be uint8, got {codes.dtype} and {scales.dtype}")
        if codes.dim() != 2 or 0 in codes.shape or codes.shape[1] % 32:
            raise ValueError(f"{name}: codes must be [n, k] with whole blocks of 32 channels, got {tuple(codes.shape)}")
        _abi.mx8_scale_rows(name, codes, scales)
        if bias is not None:
            _no_gradient(bias)
            if bias.shape != codes.shape[:1]:
                raise ValueError(f"{name}: bias {tuple(bias.shape)} does not go with {codes.shape[0]} outputs")
            bias = bias.detach().float()
        self.out_features, self.in_features = codes.shape
        self.register_buffer("codes", codes.contiguous())
        self.register_buffer("scales", scales.contiguous())
        self.register_buffer("bias", bias)

    @classmethod
    @torch.no_grad()
    def from_linear(cls, lin: torch.nn.Linear) -> MX8Linear:
        """lin in 8 bits (quantize_weight), its bias kept."""
        return cls(*quantize_weight(lin.weight.detach()), None if lin.bias is None else lin.bias.detach())

    def _apply(self, fn, recurse: bool = True):
        """Moves as any module's; a cast of the types (module.to(torch.bfloat16)) leaves the bias in float32, as the product
        takes it and with the bits that it has."""
        bias = self.bias
        super()._apply(fn, recurse)
        if bias is not None and self.bias.dtype != torch.float32:
            self.bias = bias.to(self.bias.device)
        return self

    def extra_repr(self) -> str:
        return f"in_features={self.in_features}, out_features={self.out_features}, bias={self.bias is not None}"

    def weight_values(self, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
        """The weight that the codes stand for."""
        return dequantize(Quantized(self.codes, self.scales), dtype)

    def forward(self, x, activation: str | None = None, residual: torch.Tensor | None = None,
                out: torch.Tensor | None = None) -> torch.Tensor:
        """activation(x w^T + bias) + residual in bf16. x: Quantized rows, or float rows that are quantized first.
        activation: "relu", "silu", "gelu" (by erf) or None. residual: bf16 of the output's shape; it may be out."""
        if isinstance(x, torch.Tensor):
            x = quantize(x)
        _no_gradient(residual, out)
        held = self._buffers
        return _abi.linear_mx8(x[0], x[1], held["codes"], held["scales"], held["bias"], activation, residual, out)


_module = torch.nn.modules.module
_HOOKS = ("_forward_hooks", "_forward_pre_hooks", "_backward_hooks", "_backward_pre_hooks")


def _only_the_product(lin) -> bool:
    """Whether calling lin is the product alone: no bias, hooks or forward of its own."""
    own = lin.__dict__
    return (type(lin) is MX8Linear and "forward" not in own and own["_buffers"]["bias"] is None
            and not any(own[h] for h in _HOOKS) and not _module._global_forward_hooks
            and not _module._global_forward_pre_hooks)


def _one_launch(w0, s0, w1, s1) -> bool:
    """Whether both weights' scales cover as many rows (a weight of one row goes with any)."""
    n0, n1 = w0.shape[0], w1.shape[0]
    return n0 == 1 or n1 == 1 or (s0.shape[0] == n0) == (s1.shape[0] == n1)


def linear_pair(lin0: MX8Linear, lin1: MX8Linear, x):
    """(lin0(x), lin1(x)) in one launch where both are plain products (no bias, no hooks) with scales of one kind; x as
    MX8Linear takes it, quantized once."""
    if isinstance(x, torch.Tensor):
        x = quantize(x)
    a, b = lin0._buffers, lin1._buffers
    if _only_the_product(lin0) and _only_the_product(lin1) and _one_launch(a["codes"], a["scales"], b["codes"], b["scales"]):
        return _abi.linear_mx8_pair(x[0], x[1], a["codes"], a["scales"], b["codes"], b["scales"])
    return lin0(x), lin1(x)
