"""Group norm over channels-last rows, with SiLU or without, and its forms that hand quantised rows to a Linear.

SDXL's transformer blocks put a GroupNorm in front of ``proj_in`` as FLUX's put an adaLN in front of the feed-forward
(``ops.adaln_quant_rows``); image-token rows [B, T, C] (or [B, H, W, C]) keep a token's channels together, so the norm works
on them without a transposition:

    z[b,t,c] = act((x[b,t,c] - mean[b,g]) / sqrt(var[b,g] + eps) * weight[c] + bias[c])

Statistics and arithmetic are fp32, the result is rounded once (SiLU of z below -41.6, which lies between -4e-17 and 0, comes out as
-3.6e-17).  CUDA tensors only (AssertionError otherwise); there is no
gradient: tensors that autograd follows raise RuntimeError.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import ops
from .fp4_exec import DEFAULT_FORMAT, Fp4Rows, quant_rows_fp4
from .int8_exec import _eager, quant_rows


def group_norm_rows(x: torch.Tensor, groups: int, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
                    eps: float = 1e-6, act: Optional[str] = None) -> torch.Tensor:
    """x [B, ..., C] bf16/fp16, channels last -> normed rows of the same shape and type.  ``act``: None or "silu".
    weight / bias [C] in x's type or fp32, or None.  C % 8 == 0, C <= 8192, C % groups == 0, B <= 65535."""
    assert x.is_cuda
    if _eager():
        return ops._group_norm_impl(x, groups, weight, bias, eps, act)
    ops.check_group_norm_act(act)                     # the operator knows SiLU or nothing
    return torch.ops.pq_b200.group_norm_rows(x, groups, weight, bias, eps, act == "silu")


def group_norm_quant_rows(x: torch.Tensor, groups: int, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
                          eps: float = 1e-6, act: Optional[str] = None,
                          want_normed: bool = False) -> Tuple[torch.Tensor, torch.Tensor, Optional[torch.Tensor]]:
    """(q, s, z) with z = group_norm_rows(x, ...) and (q, s) = quant_rows of z's rows; z is None unless ``want_normed``.  One
    launch where the rows fit into the GPU's shared memory (about 29 MB) and C % 16 == 0, two otherwise; the same codes."""
    assert x.is_cuda
    if _eager():
        r = ops.group_norm_quant_rows_fused(x, groups, weight, bias, eps, act, want_normed)
        if r is not None:
            return r
    z = group_norm_rows(x, groups, weight, bias, eps, act)
    q, s = quant_rows(z.reshape(-1, z.shape[-1]))
    return q, s, z if want_normed else None


def group_norm_quant_fp4(x: torch.Tensor, groups: int, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
                         eps: float = 1e-6, act: Optional[str] = None, fmt: str = DEFAULT_FORMAT) -> Fp4Rows:
    """quant_rows_fp4 of the rows of group_norm_rows(x, ...), C % 32 == 0; launches as group_norm_quant_rows."""
    assert x.is_cuda
    if _eager():
        r = ops.group_norm_quant_fp4_fused(x, groups, weight, bias, eps, act, fmt)
        if r is not None:
            return Fp4Rows(*r)
    z = group_norm_rows(x, groups, weight, bias, eps, act)
    return quant_rows_fp4(z.reshape(-1, z.shape[-1]), fmt)
