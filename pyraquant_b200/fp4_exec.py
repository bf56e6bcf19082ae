"""Linears in microscaled 4-bit floating point: both operands as E2M1 codes with block scales that the tensor cores apply.

The reference keeps 4-bit weights for storage only and expands them to INT8 (deploy/run_flux_latency.py:16-18); this module
is the 4-bit counterpart of ``int8_exec``: ``quant_rows_fp4`` and ``fp4_gemm`` beside ``quant_rows`` and
``int8_gemm_fused``, ``Fp4Linear`` beside ``Int8Linear``, ``convert_linears_to_fp4`` beside ``convert_linears_to_int8``.

Two formats (``fmt``)
  ``"mx"``  one power of two (E8M0) per 32 elements;
  ``"nv"``  one E4M3 scale per 16 elements under a power of two per row: finer scales, 6 % more bytes.
Packed rows are an ``Fp4Rows``: codes uint8 [M, K/2], scale bytes uint8 [ceil(M/128), tiles, 512] in the order the tensor cores
read them (``include/pq_b200.h`` spells it out), and the nv format's row scales fp32 [M].

CUDA tensors only; a CPU tensor raises AssertionError.  There is no gradient: the results of a quantisation are codes.
"""
from __future__ import annotations

from typing import Callable, Dict, NamedTuple, Optional, Tuple

import torch
import torch.nn as nn

from . import ops
from .int8_exec import LOWRANK_A_ATTR, LOWRANK_B_ATTR, LowRankFactors, _eager, is_bf16_whitelisted

FORMATS = tuple(ops.FP4_FORMATS)
DEFAULT_FORMAT = "nv"


class Fp4Rows(NamedTuple):
    """Packed rows: E2M1 codes, block scales and, for the nv format, row scales."""
    codes: torch.Tensor
    scales: torch.Tensor
    row_scale: Optional[torch.Tensor] = None

    @property
    def fmt(self) -> str:
        return "mx" if self.row_scale is None else "nv"


# --------------------------------------------------------------------------- operator wrappers
def quant_rows_fp4(x2: torch.Tensor, fmt: str = DEFAULT_FORMAT) -> Fp4Rows:
    """[M,K] bf16/fp16 -> packed rows; K % 32 == 0; rows may be strided (no copy when they start on 32-byte borders)."""
    assert x2.dim() == 2 and x2.is_cuda
    if _eager():
        return Fp4Rows(*ops._quant_rows_fp4_impl(x2, fmt))
    codes, scales, row = torch.ops.pq_b200.quant_rows_fp4(x2, fmt)
    return Fp4Rows(codes, scales, row if fmt == "nv" else None)


def dequant_rows_fp4(q: Fp4Rows, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The values packed rows stand for, [M,K] in ``dtype``.  bf16 holds them exactly; fp16 rounds what lies below its
    normal range.  What passes the type's largest value, by a scale that was rounded up, is clipped to it."""
    if _eager():
        return ops._dequant_rows_fp4_impl(q.codes, q.scales, q.row_scale, dtype)
    return torch.ops.pq_b200.dequant_rows_fp4(q.codes, q.scales, q.row_scale, ops.dtype_code(dtype))


def fp4_gemm(xq: Fp4Rows, w: Fp4Rows, bias: Optional[torch.Tensor] = None, out_dtype: torch.dtype = torch.bfloat16,
             lowrank: Optional[Tuple[torch.Tensor, torch.Tensor]] = None) -> torch.Tensor:
    """x [M,K] times the transpose of w [N,K] (+ fp32 bias [N]) in ``out_dtype``; both operands in the same format.
    ``lowrank``: the factors of a rank-32 term that is added before the one rounding, as ``lowrank_rows`` and
    ``lowrank_weight`` make them for these operands."""
    t, lb = lowrank if lowrank is not None else (None, None)
    if _eager():
        return ops._fp4_gemm_impl(xq.codes, xq.scales, xq.row_scale, w.codes, w.scales, w.row_scale, bias, out_dtype, t, lb)
    return torch.ops.pq_b200.fp4_gemm(xq.codes, xq.scales, xq.row_scale, w.codes, w.scales, w.row_scale, bias,
                                      ops.dtype_code(out_dtype), t, lb)


def lowrank_rows(t: torch.Tensor, xq: Fp4Rows) -> torch.Tensor:
    """Low-rank activations t [M,32] bf16/fp16 in the units of the rows they go with: fp32, t over the row scale."""
    if _eager():
        return ops._fp4_lowrank_rows_impl(t, xq.row_scale)
    return torch.ops.pq_b200.fp4_lowrank_rows(t, xq.row_scale)


def lowrank_weight(B: torch.Tensor, w: Fp4Rows) -> torch.Tensor:
    """The up-projection B [32,N] bf16/fp16 in the units of the weights it goes with: fp32 [N,32].  Plain tensor arithmetic, for
    factors that are laid out once; ``lowrank_factors`` lays B out on every call."""
    assert B.dim() == 2 and B.shape == (32, w.codes.shape[0]) and B.dtype in ops._DT
    b = B.t().float()
    return (b if w.row_scale is None else b / w.row_scale[:, None]).contiguous()


def lowrank_factors(t: torch.Tensor, xq: Fp4Rows, B: torch.Tensor, w: Fp4Rows) -> Tuple[torch.Tensor, torch.Tensor]:
    """``(lowrank_rows(t, xq), lowrank_weight(B, w))`` in one launch: what ``fp4_gemm`` takes as ``lowrank``."""
    assert B.dim() == 2 and B.shape == (32, w.codes.shape[0]), (tuple(B.shape), w.codes.shape[0])
    if _eager():
        return ops._fp4_lowrank_factors_impl(t, xq.row_scale, B, w.row_scale)
    return lowrank_rows(t, xq), lowrank_weight(B, w)


def fp4_linear_2d(x2: torch.Tensor, w: Fp4Rows, bias: Optional[torch.Tensor] = None) -> torch.Tensor:
    """x2 [M,K] -> [M,N] in x2's dtype: quantisation in the weights' format, then the product."""
    return fp4_gemm(quant_rows_fp4(x2, w.fmt), w, bias, x2.dtype)


# --------------------------------------------------------------------------- weights
def quantize_weight_fp4(w: torch.Tensor, fmt: str = DEFAULT_FORMAT) -> Fp4Rows:
    """Packed rows of a weight matrix [N,K] of any floating type, K % 32 == 0.  Plain tensor arithmetic (done once per
    layer, on any device); for 16-bit weights the bytes are those of ``quant_rows_fp4``."""
    block = ops.FP4_BLOCK.get(fmt)
    if block is None:
        ops._fp4_code(fmt)
    N, K = w.shape
    assert K > 0 and K % 32 == 0, f"K={K} must be a multiple of 32"
    b = w.detach().float().reshape(N, K // block, block)
    assert bool(torch.isfinite(b).all()), "weights must be finite"
    amax = b.abs().amax(dim=2)
    row = None
    if fmt == "mx":
        scale = (torch.frexp(amax)[1] - 3).clamp(-127, 127)                     # floor(log2) - 2; frexp's m is in [1/2, 1)
        scale = torch.where(amax > 0, scale, torch.full_like(scale, -127))
        q = torch.ldexp(b, -scale[:, :, None])
        byte = (scale + 127).to(torch.uint8)
    else:
        m, e = torch.frexp(amax.amax(dim=1))
        e = torch.where(m > 2688 / 4096, e - 11, e - 12).clamp(min=-100)
        row = torch.ldexp(torch.ones_like(m), torch.where(m > 0, e, torch.zeros_like(e)))
        s8 = (amax / row[:, None] / 6).to(torch.float8_e4m3fn)
        s = s8.float()[:, :, None]
        q = torch.where(s > 0, b / row[:, None, None] / s.clamp_min(2.0 ** -9), torch.zeros_like(b))
        byte = s8.view(torch.uint8)
    a = q.abs()
    # the borders between 0, 1/2, 1, 3/2, 2, 3, 4, 6; a value on a border goes to the even code
    code = ((a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0))
    code = (code | (torch.signbit(q).to(torch.uint8) << 3)).reshape(N, K)
    codes = (code[:, 0::2] | (code[:, 1::2] << 4)).contiguous()
    groups, tiles, _ = ops.fp4_scale_shape(N, K, fmt)
    flat = torch.zeros((groups * 128, tiles * 4), dtype=torch.uint8, device=w.device)
    flat[:N, : K // block] = byte
    scales = flat.reshape(groups, 4, 32, tiles, 4).permute(0, 3, 2, 1, 4).reshape(groups, tiles, 512).contiguous()
    return Fp4Rows(codes, scales, row)


# --------------------------------------------------------------------------- module
class Fp4Linear(LowRankFactors, nn.Module):
    """4-bit stand-in for ``nn.Linear``: packed weights held as buffers, activations quantised per call in the same
    format.  A low-rank branch (``lowrank=(A, B)`` or the ``_lowrank_A`` / ``_lowrank_B`` attributes that
    ``Int8Linear`` reads too), ``y += (x @ A) @ B`` with x @ A rounded to the activation type, is added in the product's fp32
    accumulator for rank 32 and factors in bf16 / fp16, in the activation type after the product otherwise.
    Needs in_features % 32 == 0."""

    def __init__(self, lin: nn.Linear, device: Optional[torch.device] = None, fmt: str = DEFAULT_FORMAT,
                 lowrank: Optional[Tuple[torch.Tensor, torch.Tensor]] = None):
        super().__init__()
        w = lin.weight.detach()
        if device is not None:
            w = w.to(device, non_blocking=False)
        q = quantize_weight_fp4(w, fmt)
        self.fmt = fmt
        self.register_buffer("weight_codes", q.codes)
        self.register_buffer("weight_scales", q.scales)
        self.register_buffer("weight_row_scale", q.row_scale)
        if lin.bias is not None:
            b = lin.bias.detach().float()
            self.register_buffer("bias", (b.to(device) if device is not None else b).contiguous())
        else:
            self.bias = None
        self.in_features = int(lin.in_features)
        self.out_features = int(lin.out_features)
        A, B = lowrank if lowrank is not None else (getattr(lin, LOWRANK_A_ATTR, None), getattr(lin, LOWRANK_B_ATTR, None))
        if A is not None and B is not None:
            if device is not None:
                A, B = A.to(device), B.to(device)
            self.register_buffer("lr_A", A.contiguous())
            self.register_buffer("lr_B", B.contiguous())
        else:
            self.lr_A = None
            self.lr_B = None

    @property
    def weight_rows(self) -> Fp4Rows:
        return Fp4Rows(self.weight_codes, self.weight_scales, self.weight_row_scale)

    def _apply(self, fn, recurse=True):
        """``.half()`` / ``.to(dtype)`` convert floating buffers; row scales and bias move with them but stay the fp32 they
        were (a row scale can lie outside fp16's range)."""
        keep = {n: getattr(self, n) for n in ("weight_row_scale", "bias")}
        super()._apply(fn, recurse)
        for name, v in keep.items():
            new = getattr(self, name)
            if v is not None and new.dtype != v.dtype:
                setattr(self, name, v.to(new.device))
        return self

    def _lr_At(self) -> torch.Tensor:
        """lr_A transposed, on every call like lr_B: this layer keeps nothing that a write to its buffers could leave behind."""
        return ops.lowrank_layout(self.lr_A, None)[0] if _eager() else self.lr_A.t().contiguous()

    def _with_branch(self, x2: torch.Tensor) -> torch.Tensor:
        xq, w = quant_rows_fp4(x2, self.fmt), self.weight_rows
        t = self._down(x2).to(x2.dtype)
        if t.shape[1] == 32 and self.lr_B.dtype in ops._DT:
            return fp4_gemm(xq, w, self.bias, x2.dtype, lowrank_factors(t, xq, self.lr_B, w))
        y = fp4_gemm(xq, w, self.bias, x2.dtype)
        return y.addmm_(t, self.lr_B.to(y.dtype))

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        shape = x.shape
        assert shape[-1] == self.in_features, (tuple(shape), self.in_features)
        x2 = x.detach().reshape(-1, shape[-1])                 # no gradient, not even through the low-rank branch alone
        y2 = fp4_linear_2d(x2, self.weight_rows, self.bias) if self.lr_A is None else self._with_branch(x2)
        return y2.reshape(*shape[:-1], self.out_features)

    def forward_group_norm(self, h: torch.Tensor, groups: int, weight: Optional[torch.Tensor], bias: Optional[torch.Tensor],
                           eps: float = 1e-6, act: Optional[str] = None) -> torch.Tensor:
        """``self(act(GroupNorm(h)))`` for channels-last rows h [B, ..., K], the same values as
        ``norm_exec.group_norm_rows`` followed by the layer."""
        from . import norm_exec
        K = h.shape[-1]
        assert K == self.in_features, (tuple(h.shape), self.in_features)
        if self.lr_A is not None:                              # the branch reads the 16-bit rows
            return self.forward(norm_exec.group_norm_rows(h, groups, weight, bias, eps, act))
        xq = norm_exec.group_norm_quant_fp4(h, groups, weight, bias, eps, act, self.fmt)
        return fp4_gemm(xq, self.weight_rows, self.bias, h.dtype).reshape(*h.shape[:-1], self.out_features)

    def extra_repr(self) -> str:
        return f"in={self.in_features}, out={self.out_features}, 4-bit {self.fmt} W and A, sm_100a tcgen05 kernel"


# --------------------------------------------------------------------------- model conversion
def convert_linears_to_fp4(model: nn.Module, device: Optional[str] = "cuda", fmt: str = DEFAULT_FORMAT,
                           whitelist: Callable[[str], bool] = is_bf16_whitelisted) -> Dict[str, object]:
    """Swaps every non-whitelisted ``nn.Linear`` whose in_features the format takes for ``Fp4Linear`` in place and returns
    statistics as ``convert_linears_to_int8`` does (``n_fp4_linear``, ``params_fp4``, the kept layers)."""
    dev = torch.device(device) if device is not None else None
    stats = {"n_fp4_linear": 0, "n_bf16_linear_kept": 0, "params_fp4": 0, "params_bf16_linear_kept": 0, "bf16_kept_names": []}
    for name, lin in [(n, m) for n, m in model.named_modules() if isinstance(m, nn.Linear)]:
        if whitelist(name) or lin.in_features % 32 != 0:
            stats["n_bf16_linear_kept"] += 1
            stats["params_bf16_linear_kept"] += lin.weight.numel()
            stats["bf16_kept_names"].append(name)
            continue
        parent_name, _, attr = name.rpartition(".")
        parent = model.get_submodule(parent_name) if parent_name else model
        setattr(parent, attr, Fp4Linear(lin, device=dev, fmt=fmt))
        stats["n_fp4_linear"] += 1
        stats["params_fp4"] += lin.weight.numel()
    if dev is not None and dev.type == "cuda":
        torch.cuda.synchronize()
    per = 0.5 + 1.0 / ops.FP4_BLOCK[fmt]                                         # bytes per weight
    stats["fp4_weight_gib"] = stats["params_fp4"] * per / 2**30
    stats["bf16_equiv_gib"] = stats["params_fp4"] * 2 / 2**30
    return stats
