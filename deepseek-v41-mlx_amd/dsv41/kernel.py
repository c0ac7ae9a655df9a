"""Drop-in for the native ``kernel`` module that DeepSeek's reference model imports
(docs/reference/model.py:12-19; its TileLang wrappers live in docs/reference/kernel.py).

The reference's own tests replace that module by ``sys.modules["kernel"] = kernel_stub``
(tests/test_parity.py:57-58); this module fills the same seam with the gfx950 kernels:

    import sys, dsv41.kernel
    sys.modules["kernel"] = dsv41.kernel

Covered (the attention path): the in-place QAT round trips of ``act_quant`` /
``fp4_act_quant``, ``sparse_attn``, and the 8-bit projections: ``act_quant`` to codes and scales and
``fp8_gemm``, in the release's form (blocks of 32 channels, weight blocks of 32 x 32, ue8m0 scales).
``fp4_gemm`` (the experts') and the hyper-connection Sinkhorn are outside the attention path and
raise, like the reference's test stub (tests/kernel_stub.py:127-134).
"""

from __future__ import annotations

import torch

from . import _abi


def act_quant(x: torch.Tensor, block_size: int = 128, scale_fmt=None, scale_dtype=None,
              inplace: bool = False):
    """kernel.py:98-124 with power-of-two scales (``scale_fmt="ue8m0"``): the fused quant->dequant form
    (``inplace=True``), or the e4m3 codes of x and their e8m0 scales, one per 32 channels, as fp8_gemm takes them."""
    if scale_fmt is None:
        raise NotImplementedError("dsv41.kernel.act_quant implements power-of-two (ue8m0) scales only")
    if inplace:
        _abi.fq_fp8_ue8m0(x, block_size, out=x)
        return x
    if block_size != 32 or scale_dtype not in (None, torch.float8_e8m0fnu):
        raise NotImplementedError("dsv41.kernel.act_quant gives codes in blocks of 32 with e8m0 scales only")
    codes, scales = _abi.quant_mx8(x)
    return codes.view(torch.float8_e4m3fn), scales.view(torch.float8_e8m0fnu)


def fp8_gemm(a: torch.Tensor = None, a_s: torch.Tensor = None, b: torch.Tensor = None, b_s: torch.Tensor = None,
             scale_dtype=torch.float8_e8m0fnu) -> torch.Tensor:
    """kernel.py:277-307: a [..., k] b [n, k]^T in bf16 from e4m3 codes and e8m0 scales, a_s [..., k/32] and
    b_s [ceil(n/32), k/32] (act_quant's and the release's blocks)."""
    if a is None or a_s is None or b is None or b_s is None:
        raise RuntimeError("fp8_gemm: codes and scales of both operands are needed")
    if scale_dtype is not torch.float8_e8m0fnu or not a_s.dtype == b_s.dtype == torch.float8_e8m0fnu:
        raise NotImplementedError("dsv41.kernel.fp8_gemm implements e8m0 scales only")
    if not a.dtype == b.dtype == torch.float8_e4m3fn:
        raise ValueError(f"fp8_gemm: operands must be float8_e4m3fn, got {a.dtype} and {b.dtype}")
    return _abi.linear_mx8(*(t.view(torch.uint8) for t in (a, a_s, b, b_s)))


def fp4_act_quant(x: torch.Tensor, block_size: int = 32, inplace: bool = False,
                  scale_dtype=torch.float8_e8m0fnu):
    """kernel.py:184-204: e8m0 (power-of-two) scales, or e4m3 scales (compressed KV)."""
    if not inplace:
        raise NotImplementedError("dsv41.kernel.fp4_act_quant implements the inplace round trip only")
    if scale_dtype == torch.float8_e4m3fn:
        _abi.fq_fp4_e4m3(x, block_size, out=x)
    else:
        _abi.fq_fp4_ue8m0(x, block_size, out=x)
    return x


def sparse_attn(q: torch.Tensor, kv: torch.Tensor, attn_sink: torch.Tensor, topk_idxs: torch.Tensor,
                softmax_scale: float) -> torch.Tensor:
    """kernel.py:392-403 (no head padding needed: partial head tiles are masked in-kernel)."""
    return _abi.sparse_attn(q.contiguous(), kv.contiguous(), attn_sink.float().contiguous(),
                            topk_idxs.to(torch.int32).contiguous(), softmax_scale)


def _outside_path(name):
    def f(*args, **kwargs):
        raise RuntimeError(f"{name} is outside the attention path; dsv41 does not implement it")
    return f


fp4_gemm = _outside_path("fp4_gemm")
hc_split_sinkhorn = _outside_path("hc_split_sinkhorn")
