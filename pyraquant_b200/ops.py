"""Torch-facing operators over the C ABI: each one allocates its outputs with torch, passes raw device
pointers and torch's current CUDA stream to libpq_b200.so, and is registered as a torch custom op
(namespace ``pq_b200``) with a fake implementation for shape propagation.

CUDA tensors only: a CPU tensor raises AssertionError, as the reference's ``quant_rows`` does
(deploy/int8_exec.py:221).  There is no fallback implementation.
"""
from __future__ import annotations

import ctypes
from typing import Dict, Optional, Sequence, Tuple

import torch

from . import _lib

Tensor = torch.Tensor

_DT = {torch.bfloat16: _lib.DTYPE_BF16, torch.float16: _lib.DTYPE_FP16}
# rank-32 term of the fused GEMM: tcgen05 tensor cores (True) or warp-level mma.sync in the epilogue (False)
LOWRANK_ON_TENSOR_CORES = True
# epilogue variants of pq_int8_gemm_ex
EPI_ACCUMULATE = 1      # out += y (both rounded to the output type first)
EPI_GELU_TANH = 2       # out = gelu_tanh(y rounded to the output type)
MAX_OUT_MORE = 7        # further output buffers of pq_int8_gemm_bcast
_status_words: Dict[int, Tensor] = {}


def _dt(dtype: torch.dtype) -> int:
    try:
        return _DT[dtype]
    except KeyError:
        raise TypeError(f"pq_b200 supports bfloat16 and float16, got {dtype}") from None


def _stream(t: Tensor) -> int:
    """Raw handle of torch's current stream on the tensor's device (the cheap private accessor when it exists)."""
    idx = t.device.index
    try:
        return torch._C._cuda_getCurrentRawStream(idx)
    except AttributeError:                      # pragma: no cover
        return torch.cuda.current_stream(t.device).cuda_stream


# whether the current stream records a graph (without torch.cuda's check that CUDA is initialised)
capturing = getattr(torch._C, "_cuda_isCurrentStreamCapturing", None) or torch.cuda.is_current_stream_capturing


# torch.cuda.current_device() without its check that CUDA is initialised (a tensor of the device exists already)
_current_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device


class _on_device:
    """`with torch.cuda.device(...)` only when the tensor lives on another device than the current one: the
    context manager costs several microseconds, which matters for the small 1K-stage layers."""
    __slots__ = ("ctx",)

    def __init__(self, t: Tensor):
        self.ctx = None if t.get_device() == _current_device() else torch.cuda.device(t.device)

    def __enter__(self):
        if self.ctx is not None:
            self.ctx.__enter__()

    def __exit__(self, *a):
        if self.ctx is not None:
            self.ctx.__exit__(*a)


def _ptr(t: Optional[Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


def _written_in_place(t: Tensor) -> None:
    """The library writes through raw pointers, which torch cannot see: tell it that `t` changed, so that anything
    keyed on the tensor's version counter (autograd's saved-tensor check, SharedInputGroup's cache) notices."""
    if not t.is_inference():
        torch.autograd.graph.increment_version(t)


def tensor_version(t: Tensor) -> int:
    """Version counter of `t`, or -1 for inference tensors (which do not keep one)."""
    return -1 if t.is_inference() else t._version


_lib_handle = None


def _LIB():
    global _lib_handle
    if _lib_handle is None:
        _lib_handle = _lib.load()
    return _lib_handle


_bind_handle = None


def _BIND():
    """The one-step calls of csrc/bind.cpp; each returns None for operands that need the steps written out here."""
    global _bind_handle
    if _bind_handle is None:
        _bind_handle = _lib.binding()
    return _bind_handle


def status_word(device: torch.device) -> Tensor:
    """Per-device workspace whose word 0 the GEMM kernels set when a bounded wait gives up."""
    idx = device.index if device.index is not None else torch.cuda.current_device()
    w = _status_words.get(idx)
    if w is None:
        w = torch.zeros(_lib.GEMM_WORKSPACE_BYTES // 4, dtype=torch.int32, device=torch.device("cuda", idx))
        _status_words[idx] = w
    return w


def check_device_status(device=None, clear: bool = True) -> None:
    """Synchronises and raises RuntimeError if any GEMM launched so far on `device` gave up a wait."""
    dev = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
    w = status_word(dev)
    raw = ctypes.c_int32(0)
    with torch.cuda.device(dev):
        rc = _lib.load().pq_read_status_word(w.data_ptr(), ctypes.byref(raw), int(clear),
                                             torch.cuda.current_stream(dev).cuda_stream)
    if rc == _lib.PQ_ERR_TIMEOUT:
        raise RuntimeError(f"pq_b200: a device-side wait gave up (status word 0x{raw.value & 0xffffffff:08x})")
    _lib.check(rc, "pq_read_status_word")


def _rows_ok(x2: Tensor) -> Tensor:
    """Row-strided views are consumed in place; anything the kernels cannot address is made contiguous."""
    assert x2.dim() == 2 and x2.is_cuda
    if x2.stride(1) != 1 or (x2.shape[0] > 1 and x2.stride(0) % 8 != 0) or x2.data_ptr() % 16 != 0:
        x2 = x2.contiguous()
    return x2


# ------------------------------------------------------------------------------------------------ quantisation
def _quant_rows_impl(x2: Tensor) -> Tuple[Tensor, Tensor]:
    x2 = _rows_ok(x2)
    M, K = x2.shape
    q = torch.empty((M, K), dtype=torch.int8, device=x2.device)
    s = torch.empty((M,), dtype=torch.float32, device=x2.device)
    ld = x2.stride(0) if M > 1 else max(K, x2.stride(0))
    with _on_device(x2):
        rc = _LIB().pq_quant_rows(x2.data_ptr(), _dt(x2.dtype), M, K, ld, q.data_ptr(), s.data_ptr(), _stream(x2))
    if rc:
        _lib.check(rc, f"pq_quant_rows(M={M}, K={K})")
    return q, s


def _quant_rows_g32_impl(x2: Tensor) -> Tuple[Tensor, Tensor]:
    x2 = _rows_ok(x2)
    M, K = x2.shape
    assert K % 32 == 0, K
    q = torch.empty((M, K), dtype=torch.int8, device=x2.device)
    s = torch.empty((M, K // 32), dtype=torch.float32, device=x2.device)
    ld = x2.stride(0) if M > 1 else max(K, x2.stride(0))
    with _on_device(x2):
        rc = _LIB().pq_quant_rows_g32(x2.data_ptr(), _dt(x2.dtype), M, K, ld, q.data_ptr(), s.data_ptr(),
                                           _stream(x2))
    _lib.check(rc, f"pq_quant_rows_g32(M={M}, K={K})")
    return q, s


def cat_sources_ok(x0: Tensor, x1: Tensor) -> bool:
    """Whether the two-source entry points take x0 / x1 as they are (the seam on a 64-element boundary, rows up to
    16384 elements, aligned row-strided views)."""
    def ok(t):
        return (t.dim() == 2 and t.is_cuda and t.stride(1) == 1 and (t.shape[0] <= 1 or t.stride(0) % 8 == 0)
                and t.data_ptr() % 16 == 0)
    return (ok(x0) and ok(x1) and x0.dtype == x1.dtype and x0.dtype in _DT and x0.shape[0] == x1.shape[0]
            and x0.device == x1.device and x0.shape[1] % 64 == 0 and x1.shape[1] % 8 == 0
            and x0.shape[1] + x1.shape[1] <= 16384)


def quant_rows_cat(x0: Tensor, x1: Tensor) -> Tuple[Tensor, Tensor]:
    """quant_rows(torch.cat([x0, x1], 1)) without the concatenated tensor (pq_quant_rows_cat)."""
    assert cat_sources_ok(x0, x1)
    M, K0 = x0.shape
    K1 = x1.shape[1]
    q = torch.empty((M, K0 + K1), dtype=torch.int8, device=x0.device)
    s = torch.empty((M,), dtype=torch.float32, device=x0.device)
    with _on_device(x0):
        rc = _LIB().pq_quant_rows_cat(x0.data_ptr(), K0, x0.stride(0) if M > 1 else max(K0, x0.stride(0)), x1.data_ptr(), K1,
                                      x1.stride(0) if M > 1 else max(K1, x1.stride(0)), _dt(x0.dtype), M, q.data_ptr(),
                                      s.data_ptr(), _stream(x0))
    if rc:
        _lib.check(rc, f"pq_quant_rows_cat(M={M}, K={K0}+{K1})")
    return q, s


def lowrank_down_cat(x0: Tensor, x1: Tensor, a_t: Tensor) -> Tensor:
    """lowrank_down(torch.cat([x0, x1], 1), a_t) without the concatenated tensor (pq_lowrank_down_cat)."""
    assert cat_sources_ok(x0, x1)
    M, K0 = x0.shape
    K1 = x1.shape[1]
    R = a_t.shape[0]
    assert R in LOWRANK_DOWN_COLS and a_t.dtype == x0.dtype and a_t.shape == (R, K0 + K1) and a_t.is_contiguous()
    t = torch.empty((M, R), dtype=x0.dtype, device=x0.device)
    ws = status_word(x0.device)
    with _on_device(x0):
        rc = _LIB().pq_lowrank_down_cat(x0.data_ptr(), K0, x0.stride(0) if M > 1 else max(K0, x0.stride(0)), x1.data_ptr(), K1,
                                        x1.stride(0) if M > 1 else max(K1, x1.stride(0)), _dt(x0.dtype), a_t.data_ptr(),
                                        K0 + K1, R, t.data_ptr(), R, M, ws.data_ptr(), ws.numel() * 4, _stream(x0))
    if rc:
        _lib.check(rc, f"pq_lowrank_down_cat(M={M}, K={K0}+{K1})")
    return t


def adaln_quant_rows(x2: Tensor, scale: Tensor, shift: Tensor, eps: float = 1e-6, rows_per_sample: int = 0,
                     want_modulated: bool = True) -> Tuple[Tensor, Tensor, Optional[Tensor]]:
    """(q, s, z) with z = LayerNorm(x2) * (1 + scale) + shift and (q, s) = quant_rows(z), in one pass over x2
    (pq_adaln_quant_rows).  scale / shift: [K] or [samples, K]; row m belongs to sample m // rows_per_sample.
    z is None unless want_modulated."""
    x2 = _rows_ok(x2)
    M, K = x2.shape
    scale = scale.reshape(-1, K); shift = shift.reshape(-1, K)
    assert scale.shape == shift.shape and scale.dtype == x2.dtype and shift.dtype == x2.dtype, (scale.shape, shift.shape)
    assert scale.is_cuda and shift.is_cuda and K % 8 == 0 and K <= 16384, K
    samples = scale.shape[0]
    if samples == 1:
        rows_per_sample = 0
    else:
        assert rows_per_sample > 0 and samples * rows_per_sample >= M, (samples, rows_per_sample, M)
    scale = scale.contiguous(); shift = shift.contiguous()
    q = torch.empty((M, K), dtype=torch.int8, device=x2.device)
    s = torch.empty((M,), dtype=torch.float32, device=x2.device)
    z = torch.empty((M, K), dtype=x2.dtype, device=x2.device) if want_modulated else None
    ld = x2.stride(0) if M > 1 else max(K, x2.stride(0))
    with _on_device(x2):
        rc = _LIB().pq_adaln_quant_rows(x2.data_ptr(), _dt(x2.dtype), M, K, ld, scale.data_ptr(), shift.data_ptr(), K,
                                        int(rows_per_sample), float(eps), _ptr(z), K, q.data_ptr(), s.data_ptr(), _stream(x2))
    if rc:
        _lib.check(rc, f"pq_adaln_quant_rows(M={M}, K={K})")
    return q, s, z


GROUP_NORM_ACTS = {None: _lib.ACT_NONE, "silu": _lib.ACT_SILU}
GROUP_NORM_MAX_C = 8192


def _affine_vector(v: Optional[Tensor]) -> Optional[Tensor]:
    """A contiguous vector that starts on a 16-byte border."""
    if v is None or (v.dim() == 1 and v.is_contiguous() and v.data_ptr() % 16 == 0):
        return v
    return v.reshape(-1).clone(memory_format=torch.contiguous_format)


def check_group_norm_act(act: Optional[str]) -> None:
    if act not in GROUP_NORM_ACTS:
        raise ValueError(f"unknown activation {act!r} (expected one of {tuple(GROUP_NORM_ACTS)})")


def group_norm_args(x: Tensor, groups: int, weight: Optional[Tensor], bias: Optional[Tensor], act: Optional[str]):
    """Checks a group norm's operands; returns x as [B, T, C] with rows the kernels take, the affine vectors (both fp32 or both in
    x's type) and the activation's code."""
    assert x.is_cuda and x.dim() >= 2, "channels-last rows [B, ..., C] on a GPU"
    _dt(x.dtype)
    check_group_norm_act(act)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, bias)):
        raise RuntimeError("group norm has no gradient here: call it under torch.no_grad() or on detached tensors")
    C = x.shape[-1]
    assert groups > 0 and C % groups == 0, f"{C} channels in {groups} groups"
    assert C % 8 == 0 and 0 < C <= GROUP_NORM_MAX_C, f"{C} channels: a multiple of 8 up to {GROUP_NORM_MAX_C}"
    for v in (weight, bias):
        assert v is None or (v.numel() == C and v.device == x.device and v.dtype in (x.dtype, torch.float32)), \
            "weight and bias: one entry per channel, in the activation type or fp32, on the same device"
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        weight, bias = weight.float(), bias.float()
    weight, bias = _affine_vector(weight), _affine_vector(bias)
    T = 1
    for n in x.shape[1:-1]:
        T *= n
    x3 = x.reshape(x.shape[0], T, C)
    if (x3.stride(2) != 1 or x3.data_ptr() % 16 != 0 or (T > 1 and (x3.stride(1) % 8 != 0 or x3.stride(1) < C))
            or (x3.shape[0] > 1 and x3.stride(0) % 8 != 0)):
        x3 = x3.clone(memory_format=torch.contiguous_format)
    return x3, weight, bias, GROUP_NORM_ACTS[act]


def _group_norm_call(name: str, x: Tensor, groups: int, weight: Optional[Tensor], bias: Optional[Tensor], eps: float,
                     act: Optional[str], outputs):
    """Runs one of the pq_group_norm entry points on x, step by step, for what the one-step call (csrc/bind.cpp) leaves to it.
    `outputs(x3, B, T, C)` allocates and returns (result, the entry point's output arguments).  None when the entry point does
    not take the size (its rows do not fit on the chip)."""
    x3, weight, bias, code = group_norm_args(x, groups, weight, bias, act)
    B, T, C = x3.shape
    result, args = outputs(x3, B, T, C)
    if B * T == 0:
        return result
    lib = _LIB()
    f32 = (weight is not None and weight.dtype == torch.float32) or (bias is not None and bias.dtype == torch.float32)
    with _on_device(x3):
        nbytes = lib.pq_group_norm_workspace_bytes(B, T, C, groups)
        ws = x3.new_empty((nbytes,), dtype=torch.uint8)
        rc = getattr(lib, name)(x3.data_ptr(), _DT[x.dtype], B, T, C, x3.stride(1) if T > 1 else C, x3.stride(0) if B > 1 else T * C,
                                groups, _ptr(weight), _ptr(bias), int(f32), float(eps), code, *args, ws.data_ptr(), nbytes,
                                status_word(x3.device).data_ptr(), _stream(x3))
    if rc == _lib.PQ_ERR_UNSUPPORTED:
        return None
    if rc:
        _lib.check(rc, f"{name}(B={B}, T={T}, C={C}, groups={groups})")
    return result


# what csrc/bind.cpp calls the forms of the norm
_NORM_Z, _NORM_INT8, _NORM_FP4 = 0, 1, {"mx": 2, "nv": 3}


def _group_norm_bound(x: Tensor, groups: int, weight: Optional[Tensor], bias: Optional[Tensor], eps: float, act: Optional[str],
                      mode: int, want_z: bool):
    """The one-step call: its result, None for operands that need the general one, False for rows that do not fit."""
    code = GROUP_NORM_ACTS.get(act, -1)
    if code < 0 or x.dim() != 3 or not x.is_cuda:
        return None
    return _BIND().group_norm(x, groups, weight, bias, eps, code, mode, want_z, status_word(x.device).data_ptr())


def _group_norm_impl(x: Tensor, groups: int, weight: Optional[Tensor], bias: Optional[Tensor], eps: float,
                     act: Optional[str]) -> Tensor:
    out = _group_norm_bound(x, groups, weight, bias, eps, act, _NORM_Z, True)
    if out is not None:
        return out

    def outputs(x3, B, T, C):
        z = torch.empty_like(x, memory_format=torch.contiguous_format)
        return z, (z.data_ptr(), C, T * C)
    out = _group_norm_call("pq_group_norm", x, groups, weight, bias, eps, act, outputs)
    if out is None:
        raise RuntimeError(f"pq_group_norm: {groups} groups of {x.shape[-1]} channels leave no room for a row on the chip")
    return out


def group_norm_quant_rows_fused(x: Tensor, groups: int, weight: Optional[Tensor], bias: Optional[Tensor], eps: float,
                                act: Optional[str], want_normed: bool):
    """(q, s, z or None) in one launch (pq_group_norm_quant_rows), or None when the size does not fit."""
    if x.shape[-1] % 16:
        return None
    r = _group_norm_bound(x, groups, weight, bias, eps, act, _NORM_INT8, want_normed)
    if r is not None:
        return r or None

    def outputs(x3, B, T, C):
        z = torch.empty_like(x, memory_format=torch.contiguous_format) if want_normed else None
        q, s = x3.new_empty((B * T, C), dtype=torch.int8), x3.new_empty((B * T,), dtype=torch.float32)
        return (q, s, z), (_ptr(z), C, T * C, q.data_ptr(), s.data_ptr())
    return _group_norm_call("pq_group_norm_quant_rows", x, groups, weight, bias, eps, act, outputs)


def group_norm_quant_fp4_fused(x: Tensor, groups: int, weight: Optional[Tensor], bias: Optional[Tensor], eps: float,
                               act: Optional[str], fmt: str):
    """(codes, scales, row scales or None) in one launch (pq_group_norm_quant_fp4), or None when the size does not fit."""
    code = _fp4_code(fmt)
    assert x.shape[-1] % 32 == 0, f"K={x.shape[-1]} must be a multiple of 32"
    r = _group_norm_bound(x, groups, weight, bias, eps, act, _NORM_FP4[fmt], False)
    if r is not None:
        return r or None

    def outputs(x3, B, T, C):
        M = B * T
        codes = x3.new_empty((M, C // 2), dtype=torch.uint8)
        scales = x3.new_empty(fp4_scale_shape(M, C, fmt), dtype=torch.uint8)
        row = x3.new_empty((M,), dtype=torch.float32) if fmt == "nv" else None
        return (codes, scales, row), (code, codes.data_ptr(), scales.data_ptr(), _ptr(row))
    return _group_norm_call("pq_group_norm_quant_fp4", x, groups, weight, bias, eps, act, outputs)


def _gather_quant_rows_impl(canvas: Tensor, row_idx: Tensor) -> Tuple[Tensor, Tensor]:
    canvas = _rows_ok(canvas)
    assert row_idx.is_cuda and row_idx.dtype == torch.int32 and row_idx.dim() == 1 and row_idx.is_contiguous()
    rows, K = canvas.shape
    M = row_idx.numel()
    q = torch.empty((M, K), dtype=torch.int8, device=canvas.device)
    s = torch.empty((M,), dtype=torch.float32, device=canvas.device)
    with _on_device(canvas):
        rc = _LIB().pq_gather_quant_rows(canvas.data_ptr(), _dt(canvas.dtype), rows, K, max(K, canvas.stride(0)),
                                              row_idx.data_ptr(), M, q.data_ptr(), s.data_ptr(), _stream(canvas))
    _lib.check(rc, f"pq_gather_quant_rows(M={M}, K={K})")
    return q, s


def _gather_rows_impl(canvas: Tensor, row_idx: Tensor) -> Tensor:
    canvas = _rows_ok(canvas)
    assert row_idx.is_cuda and row_idx.dtype == torch.int32 and row_idx.dim() == 1 and row_idx.is_contiguous()
    rows, K = canvas.shape
    M = row_idx.numel()
    out = torch.empty((M, K), dtype=canvas.dtype, device=canvas.device)
    with _on_device(canvas):
        rc = _LIB().pq_gather_rows(canvas.data_ptr(), _dt(canvas.dtype), rows, K, max(K, canvas.stride(0)),
                                        row_idx.data_ptr(), M, out.data_ptr(), K, _stream(canvas))
    _lib.check(rc, f"pq_gather_rows(M={M}, K={K})")
    return out


# ------------------------------------------------------------------------------------------------ low-rank down-projection
# True: t = x @ lr_A runs on this library's streaming tcgen05 kernel; False: torch's matmul, as the reference does
LOWRANK_DOWN_NATIVE = True
# rows from which the library's own kernels are used: all.  Measured back to back on inputs rotating through HBM, device time
# at K = 15360 and K = 3072, us: 66048 rows 296 and 65, 16896 rows 82 and 20, 4608 rows 29 and 9.6, 512 rows 9.8 and 7.4
# (torch's cuBLAS matmul 349 and 76 at 66048 rows, 79 and 21 at 16896).
LOWRANK_DOWN_MIN_ROWS = 1
# output widths the kernel is built for: one rank-32 factor, or up to four side by side
LOWRANK_DOWN_COLS = (32, 64, 96, 128)


def lowrank_down(x2: Tensor, a_t: Tensor) -> Tensor:
    """t [M, R] = x2 [M, K] @ A [K, R] with A given transposed (a_t [R, K] contiguous; R in LOWRANK_DOWN_COLS), fp32
    accumulation, rounded to the activation dtype (pq_lowrank_down)."""
    assert x2.is_cuda and x2.dim() == 2 and x2.stride(1) == 1 and x2.dtype in _DT
    R = a_t.shape[0]
    assert R in LOWRANK_DOWN_COLS, f"{R} columns; supported: {LOWRANK_DOWN_COLS}"
    assert a_t.dtype == x2.dtype and a_t.shape == (R, x2.shape[1]) and a_t.is_contiguous() and a_t.device == x2.device
    M, K = x2.shape
    t = torch.empty((M, R), dtype=x2.dtype, device=x2.device)
    ws = status_word(x2.device)
    ld = x2.stride(0) if M > 1 else max(K, x2.stride(0))
    with _on_device(x2):
        rc = _LIB().pq_lowrank_down(x2.data_ptr(), _dt(x2.dtype), ld, a_t.data_ptr(), K, R, t.data_ptr(), R, M, K,
                                    ws.data_ptr(), ws.numel() * 4, _stream(x2))
    _lib.check(rc, f"pq_lowrank_down(M={M}, K={K})")
    return t


def lowrank_layout(A: Optional[Tensor], B: Optional[Tensor]) -> Tuple[Optional[Tensor], Optional[Tensor]]:
    """(A.t(), B.t()), contiguous, of a branch's factors A [K, R] and B [R, N] (each may be left out): one launch for CUDA factors of rank 32
    in a 16-bit type (pq_lowrank_layout), torch's copies otherwise."""
    r = _BIND().lowrank_layout(A, B) if (A if A is not None else B).is_cuda else None
    if r is not None:
        return r
    a_ok = A is None or (A.is_cuda and A.dim() == 2 and A.dtype in _DT and A.shape[1] == 32 and A.is_contiguous() and A.data_ptr() % 16 == 0)
    b_ok = B is None or (B.is_cuda and B.dim() == 2 and B.dtype in _DT and B.shape[0] == 32 and B.is_contiguous())
    if not (a_ok and b_ok) or (A is not None and B is not None and A.device != B.device):
        return (None if A is None else A.t().contiguous()), (None if B is None else B.t().contiguous())
    K, N = 0 if A is None else A.shape[0], 0 if B is None else B.shape[1]
    a_t = None if A is None else A.new_empty((32, K))
    b_t = None if B is None else B.new_empty((N, 32))
    like = A if A is not None else B
    with _on_device(like):
        rc = _LIB().pq_lowrank_layout(_ptr(A), 32, _ptr(a_t), K, _ptr(B), N, _ptr(b_t), N, _stream(like))
    if rc:
        _lib.check(rc, f"pq_lowrank_layout(K={K}, N={N})")
    return a_t, b_t


def lowrank_down_ok(x2: Tensor) -> bool:
    """Shapes pq_lowrank_down takes without a copy and is the faster choice for."""
    return (LOWRANK_DOWN_NATIVE and x2.is_cuda and x2.dtype in _DT and x2.dim() == 2 and x2.stride(1) == 1
            and x2.shape[1] % 8 == 0 and x2.stride(0) % 8 == 0 and x2.data_ptr() % 16 == 0
            and x2.shape[0] >= LOWRANK_DOWN_MIN_ROWS)


# row lengths the one-launch form (pq_quant_rows_lowrank) is used for.  Below 512 columns a block is too little work for
# its two sweeps and the exchange between them (65536 rows, one launch / two, us: 256 columns 23.0 / 19.5, 512 columns
# 29.3 / 29.4, 1536 columns 71 / 85); above 16384 a column slice of A no longer fits beside the tiles.
QUANT_LOWRANK_K = (512, 16384)


def quant_lowrank_ok(x2: Tensor) -> bool:
    """Inputs pq_quant_rows_lowrank takes without a copy and is the faster choice for."""
    return lowrank_down_ok(x2) and QUANT_LOWRANK_K[0] <= x2.shape[1] <= QUANT_LOWRANK_K[1]


def quant_rows_lowrank(x2: Tensor, a_t: Tensor, x_more: Optional[Tensor] = None) -> Tuple[Tensor, Tensor, Tensor]:
    """(q, s, t): quant_rows and lowrank_down of x2 (or of [x2 | x_more]) in one launch that reads the rows once from memory
    (pq_quant_rows_lowrank); a_t [32, K] contiguous."""
    M, K0 = x2.shape
    K1 = x_more.shape[1] if x_more is not None else 0
    K = K0 + K1
    assert x2.stride(1) == 1 and (x_more is None or cat_sources_ok(x2, x_more))
    assert a_t.dtype == x2.dtype and a_t.shape == (32, K) and a_t.is_contiguous() and a_t.device == x2.device
    dev = x2.device
    q = torch.empty((M, K), dtype=torch.int8, device=dev)
    s = torch.empty((M,), dtype=torch.float32, device=dev)
    t = torch.empty((M, 32), dtype=x2.dtype, device=dev)
    ws = status_word(dev)
    ld0 = x2.stride(0) if M > 1 else max(K0, x2.stride(0))
    ld1 = 0 if x_more is None else (x_more.stride(0) if M > 1 else max(K1, x_more.stride(0)))
    with _on_device(x2):
        rc = _LIB().pq_quant_rows_lowrank(x2.data_ptr(), K0, ld0, _ptr(x_more), K1, ld1, _dt(x2.dtype), M, a_t.data_ptr(), K, 32,
                                          q.data_ptr(), s.data_ptr(), t.data_ptr(), 32, ws.data_ptr(), ws.numel() * 4,
                                          _stream(x2))
    if rc:
        _lib.check(rc, f"pq_quant_rows_lowrank(M={M}, K={K0}+{K1})")
    return q, s, t


def linear_scratch_bytes(M: int, K: int, rank: int) -> int:
    """pq_int8_linear_scratch_bytes, computed here (a call through ctypes costs as much as the arithmetic saves)."""
    up = lambda v: (v + 255) & ~255
    return up(M * K) + up(2 * M * rank) + up(4 * M)


def linear_g32(x2: Tensor, w_int8: Tensor, s_w_gm: Tensor, bias: Optional[Tensor]) -> Optional[Tensor]:
    """Quantisation and group-32 GEMM in one call (pq_int8_linear_g32); None when an operand is not as the kernels take it."""
    M, K = x2.shape
    N = w_int8.shape[0]
    if (M == 0 or x2.stride(1) != 1 or x2.stride(0) % 8 or x2.data_ptr() % 16 or K % 128 or K > 16384 or N % 4
            or x2.dtype not in _DT or not x2.is_cuda or w_int8.device != x2.device or w_int8.shape[1] != K
            or not w_int8.is_contiguous() or w_int8.dtype != torch.int8 or s_w_gm.dtype != torch.float32
            or s_w_gm.shape != (K // 32, N) or not s_w_gm.is_contiguous()
            or (bias is not None and (bias.dtype != torch.float32 or bias.numel() != N or not bias.is_contiguous()))):
        return None
    ng = (M * (K // 32) * 4 + 255) & ~255
    nbytes = ((M * K + 255) & ~255) + ng
    scratch = x2.new_empty((nbytes,), dtype=torch.uint8)
    out = x2.new_empty((M, N))
    ws = status_word(x2.device)
    code = _DT[x2.dtype]
    with _on_device(x2):
        rc = _LIB().pq_int8_linear_g32(x2.data_ptr(), code, x2.stride(0) if M > 1 else K, w_int8.data_ptr(), K, s_w_gm.data_ptr(),
                                       _ptr(bias), scratch.data_ptr(), nbytes, out.data_ptr(), N, M, N, K, ws.data_ptr(),
                                       _lib.GEMM_WORKSPACE_BYTES, _stream(x2))
    if rc:
        _lib.check(rc, f"pq_int8_linear_g32(M={M}, N={N}, K={K})")
    return out


# ------------------------------------------------------------------------------------------------ 4-bit storage
def pack_int4(codes: Tensor) -> Tensor:
    """int8 codes in [-8, 7], shape [N, K] with K even -> uint8 [N, K/2]: element 2b in the low nibble of byte b,
    element 2b+1 in the high nibble (two's complement).  Plain tensor arithmetic: done once per layer, on any device."""
    assert codes.dtype == torch.int8 and codes.dim() == 2 and codes.shape[1] % 2 == 0
    assert int(codes.min()) >= -8 and int(codes.max()) <= 7, "codes do not fit four bits"
    u = codes.to(torch.int16) & 0xF
    return (u[:, 0::2] | (u[:, 1::2] << 4)).to(torch.uint8).contiguous()


def unpack_int4(packed: Tensor, out: Optional[Tensor] = None) -> Tensor:
    """uint8 [N, K/2] packed nibbles -> int8 [N, K] on the device (pq_unpack_int4)."""
    assert packed.is_cuda and packed.dtype == torch.uint8 and packed.dim() == 2 and packed.is_contiguous()
    N, K = packed.shape[0], packed.shape[1] * 2
    assert K % 32 == 0, f"K={K} must be a multiple of 32"
    if out is None:
        out = torch.empty((N, K), dtype=torch.int8, device=packed.device)
    assert out.shape == (N, K) and out.dtype == torch.int8 and out.is_contiguous() and out.device == packed.device
    with _on_device(packed):
        rc = _LIB().pq_unpack_int4(packed.data_ptr(), K // 2, out.data_ptr(), K, N, K, _stream(packed))
    _lib.check(rc, f"pq_unpack_int4(N={N}, K={K})")
    _written_in_place(out)
    return out


# ------------------------------------------------------------------------------------------------ 4-bit floating point
FP4_FORMATS = {"mx": _lib.FP4_MX, "nv": _lib.FP4_NV}
FP4_BLOCK = {"mx": 32, "nv": 16}                     # elements per scale


def fp4_scale_shape(M: int, K: int, fmt: str) -> Tuple[int, int, int]:
    """Shape of the scale array: [row groups of 128, scale tiles, 512 bytes]."""
    return (M + 127) // 128, (K + 4 * FP4_BLOCK[fmt] - 1) // (4 * FP4_BLOCK[fmt]), 512


def _fp4_code(fmt: str) -> int:
    try:
        return FP4_FORMATS[fmt]
    except KeyError:
        raise ValueError(f"unknown 4-bit format {fmt!r} (expected one of {tuple(FP4_FORMATS)})") from None


def fp4_rows_aligned(x2: Tensor) -> Tensor:
    """The 4-bit kernels load 32 bytes at a time: rows that start elsewhere are made contiguous, and so are rows that overlap (one
    row seen many times)."""
    assert x2.dim() == 2 and x2.is_cuda
    if (x2.stride(1) != 1 or (x2.shape[0] > 1 and (x2.stride(0) % 16 != 0 or x2.stride(0) < x2.shape[1]))
            or x2.data_ptr() % 32 != 0):
        x2 = x2.clone(memory_format=torch.contiguous_format)
    return x2


def _quant_rows_fp4_impl(x2: Tensor, fmt: str) -> Tuple[Tensor, Tensor, Optional[Tensor]]:
    code = _fp4_code(fmt)
    r = _BIND().quant_rows_fp4(x2, code)
    if r is not None:
        return r
    dt = _dt(x2.dtype)
    x2 = fp4_rows_aligned(x2)
    M, K = x2.shape
    assert K > 0 and K % 32 == 0, f"K={K} must be a multiple of 32"
    codes = x2.new_empty((M, K // 2), dtype=torch.uint8)
    scales = x2.new_empty(fp4_scale_shape(M, K, fmt), dtype=torch.uint8)
    row_scale = x2.new_empty((M,), dtype=torch.float32) if fmt == "nv" else None
    with _on_device(x2):
        rc = _LIB().pq_quant_rows_fp4(x2.data_ptr(), dt, M, K, x2.stride(0) if M > 1 else K, code, codes.data_ptr(),
                                      scales.data_ptr(), _ptr(row_scale), _stream(x2))
    if rc:
        _lib.check(rc, f"pq_quant_rows_fp4(M={M}, K={K}, {fmt})")
    return codes, scales, row_scale


def check_fp4_rows(codes: Tensor, scales: Tensor, row_scale: Optional[Tensor], what: str) -> Tuple[str, int, int]:
    """(format, rows, K) of packed rows whose parts fit together (AssertionError otherwise): the C ABI receives bare
    pointers."""
    assert codes.is_cuda and codes.dim() == 2 and codes.dtype == torch.uint8, f"{what}: codes are a uint8 matrix on a GPU"
    fmt = "mx" if row_scale is None else "nv"
    M, K = codes.shape[0], codes.shape[1] * 2
    assert K > 0 and K % 32 == 0, f"{what}: K={K} must be a positive multiple of 32"
    assert (scales.dtype == torch.uint8 and tuple(scales.shape) == fp4_scale_shape(M, K, fmt) and scales.is_contiguous()
            and scales.device == codes.device), f"{what}: scales {tuple(scales.shape)} do not fit [{M}, {K}] {fmt} rows"
    assert row_scale is None or (row_scale.dtype == torch.float32 and row_scale.numel() == M and row_scale.is_contiguous()
                                 and row_scale.device == codes.device), f"{what}: one fp32 row scale per row"
    return fmt, M, K


def _codes_aligned(codes: Tensor) -> Tensor:
    if (codes.stride(1) != 1 or (codes.shape[0] > 1 and (codes.stride(0) % 16 != 0 or codes.stride(0) < codes.shape[1]))
            or codes.data_ptr() % 16 != 0):
        codes = codes.clone(memory_format=torch.contiguous_format)
    return codes


def _dequant_rows_fp4_impl(codes: Tensor, scales: Tensor, row_scale: Optional[Tensor], dtype: torch.dtype) -> Tensor:
    dt = _dt(dtype)
    out = _BIND().dequant_rows_fp4(codes, scales, row_scale, dtype is torch.bfloat16)
    if out is not None:
        return out
    fmt, M, K = check_fp4_rows(codes, scales, row_scale, "dequant_rows_fp4")
    codes = _codes_aligned(codes)
    out = codes.new_empty((M, K), dtype=dtype)
    with _on_device(codes):
        rc = _LIB().pq_dequant_rows_fp4(codes.data_ptr(), codes.stride(0) if M > 1 else K // 2, scales.data_ptr(),
                                        _ptr(row_scale), FP4_FORMATS[fmt], out.data_ptr(), dt, K, M, K, _stream(codes))
    if rc:
        _lib.check(rc, f"pq_dequant_rows_fp4(M={M}, K={K}, {fmt})")
    return out


def _fp4_gemm_impl(xq: Tensor, xs: Tensor, x_row: Optional[Tensor], wq: Tensor, ws: Tensor, w_row: Optional[Tensor],
                   bias: Optional[Tensor], out_dtype: torch.dtype, t: Optional[Tensor] = None,
                   lb: Optional[Tensor] = None) -> Tensor:
    dt = _dt(out_dtype)
    if xq.is_cuda:
        out = _BIND().fp4_gemm(xq, xs, x_row, wq, ws, w_row, bias, out_dtype is torch.bfloat16, status_word(xq.device).data_ptr(),
                               _lib.GEMM_WORKSPACE_BYTES, t, lb)
        if out is not None:
            return out
    fmt, M, K = check_fp4_rows(xq, xs, x_row, "fp4_gemm, activations")
    fmt_w, N, K_w = check_fp4_rows(wq, ws, w_row, "fp4_gemm, weights")
    assert fmt_w == fmt and K_w == K, f"{fmt} activations with K={K}, {fmt_w} weights with K={K_w}"
    assert N > 0 and wq.device == xq.device
    assert bias is None or (bias.dtype == torch.float32 and bias.numel() == N and bias.is_contiguous()
                            and bias.device == xq.device), "bias is an fp32 vector with one entry per output channel"
    assert (t is None) == (lb is None), "a low-rank term has two factors"
    for v, rows in ((t, M), (lb, N)):
        assert v is None or (v.dtype == torch.float32 and tuple(v.shape) == (rows, 32) and v.is_contiguous() and v.device == xq.device
                             and v.data_ptr() % 16 == 0), "low-rank factors are contiguous fp32 [M, 32] and [N, 32]"
    xq = _codes_aligned(xq); wq = _codes_aligned(wq)
    out = xq.new_empty((M, N), dtype=out_dtype)
    st = status_word(xq.device)
    with _on_device(xq):
        rc = _LIB().pq_fp4_gemm_lowrank(xq.data_ptr(), xq.stride(0) if M > 1 else K // 2, xs.data_ptr(), _ptr(x_row), wq.data_ptr(),
                                        wq.stride(0) if N > 1 else K // 2, ws.data_ptr(), _ptr(w_row), _ptr(bias), _ptr(t), _ptr(lb),
                                        FP4_FORMATS[fmt], out.data_ptr(), dt, N, M, N, K, st.data_ptr(), st.numel() * 4, _stream(xq))
    if rc:
        _lib.check(rc, f"pq_fp4_gemm(M={M}, N={N}, K={K}, {fmt})")
    return out


# ------------------------------------------------------------------------------------------------ GEMM
def epilogue_supported(N: int, out_stride0: int, out_ptr: int, has_lowrank: bool, rank: int = 32) -> bool:
    """Whether pq_int8_gemm_ex takes this problem (its variants live in the CTA-pair kernel's vector stores)."""
    return N % 32 == 0 and out_stride0 % 8 == 0 and out_ptr % 16 == 0 and (not has_lowrank or rank == 32)


def check_gemm_extents(M: int, N: int, K: int, s_row: Tensor, w_scale: Tensor, bias: Optional[Tensor],
                        t: Optional[Tensor], lb: Optional[Tensor], lb_t: Optional[Tensor] = None,
                        s_lo: Optional[Tensor] = None, m_hi: Optional[int] = None) -> None:
    """The C ABI receives bare pointers, so a scale, bias or low-rank tensor that is too short would be read out of
    bounds on the device.  Every operand's extent is checked here, on the host, before anything is launched
    (AssertionError, like the reference's shape asserts)."""
    assert s_row.numel() == M, f"s_row has {s_row.numel()} entries for {M} rows"
    assert w_scale.numel() == N, f"w_scale has {w_scale.numel()} entries for {N} output channels"
    assert bias is None or bias.numel() == N, f"bias has {bias.numel()} entries for {N} output channels"
    assert s_lo is None or s_lo.numel() == N, f"low-tier scale has {s_lo.numel()} entries for {N} output channels"
    assert m_hi is None or 0 <= int(m_hi) <= M, f"m_hi={m_hi} outside [0, {M}]"
    assert (t is None) == (lb is None), "t and lb go together"
    if t is not None:
        assert t.dim() == 2 and lb.dim() == 2 and t.shape[0] == M and lb.shape == (t.shape[1], N), \
            f"low-rank operands t {tuple(t.shape)} / lb {tuple(lb.shape)} do not fit [M={M}, R] / [R, N={N}]"
        assert lb_t is None or tuple(lb_t.shape) == (N, t.shape[1]), f"lb_t {tuple(lb_t.shape)} is not [N, R]"


def _gemm_impl(xq: Tensor, s_row: Tensor, w_int8: Tensor, w_scale: Tensor, bias: Optional[Tensor],
               t: Optional[Tensor], lb: Optional[Tensor], out_dtype: torch.dtype,
               dbg_acc: Optional[Tensor] = None, w_lo: Optional[Tensor] = None, s_lo: Optional[Tensor] = None,
               m_hi: Optional[int] = None, lb_t: Optional[Tensor] = None, epilogue: int = 0,
               out: Optional[Tensor] = None, out_more: Optional[Sequence[Tensor]] = None,
               gate: Optional[Tensor] = None, gate_rows: int = 0) -> Tensor:
    assert xq.is_cuda and xq.dtype == torch.int8 and xq.dim() == 2 and xq.stride(1) == 1
    assert w_int8.dtype == torch.int8 and w_int8.dim() == 2 and w_int8.stride(1) == 1
    M, K = xq.shape
    N = w_int8.shape[0]
    assert w_int8.shape[1] == K, (w_int8.shape, K)
    assert K % 16 == 0, f"K={K} must be a multiple of 16"
    assert s_row.dtype == torch.float32 and w_scale.dtype == torch.float32
    check_gemm_extents(M, N, K, s_row, w_scale, bias, t, lb, lb_t, s_lo, m_hi if w_lo is not None else None)
    s_row = s_row.contiguous(); w_scale = w_scale.contiguous()
    if bias is not None:
        assert bias.dtype == torch.float32
        bias = bias.contiguous()
    if xq.stride(0) % 16 != 0 or xq.data_ptr() % 16 != 0:
        xq = xq.contiguous()
    if w_int8.stride(0) % 16 != 0 or w_int8.data_ptr() % 16 != 0:
        w_int8 = w_int8.contiguous()
    if out is None:
        assert not (epilogue & EPI_ACCUMULATE), "accumulation needs the tensor to add onto"
        out = torch.empty((M, N), dtype=out_dtype, device=xq.device)
    else:
        assert out.shape == (M, N) and out.dtype == out_dtype and out.stride(1) == 1 and out.device == xq.device
    R = 0
    ldt = ldb = 0
    if t is not None:
        assert lb is not None and t.dtype == out_dtype and lb.dtype == out_dtype, (t.dtype, lb.dtype, out_dtype)
        if t.stride(1) != 1 or t.stride(0) % 8 != 0 or t.data_ptr() % 16 != 0:
            t = t.contiguous()
        if lb.stride(1) != 1 or lb.stride(0) % 8 != 0 or lb.data_ptr() % 16 != 0:
            lb = lb.contiguous()
        R = t.shape[1]
        ldt, ldb = t.stride(0), lb.stride(0)
        if M == 1:
            ldt = max(ldt, R)
        if lb_t is None and R == 32 and LOWRANK_ON_TENSOR_CORES:
            lb_t = lb.t().contiguous()        # K-major copy for the tcgen05 low-rank path (callers may cache it)
        if lb_t is not None:
            assert lb_t.shape == (N, R) and lb_t.dtype == out_dtype and lb_t.is_contiguous()
    ws = status_word(xq.device)
    lib = _LIB()
    ldx = xq.stride(0) if M > 1 else max(K, xq.stride(0))
    ldo = out.stride(0) if M > 1 else max(N, out.stride(0))
    if out_more:
        # further destinations of the output stores (pq_int8_gemm_bcast): same extent, dtype and row stride as `out`;
        # they may live on other GPUs of the node (peer memory mapped into this process)
        assert w_lo is None and dbg_acc is None and len(out_more) <= MAX_OUT_MORE, len(out_more)
        assert epilogue_supported(N, ldo, out.data_ptr(), t is not None, R or 32), "shape needs the CTA-pair kernel"
        for o in out_more:
            assert o.shape == (M, N) and o.dtype == out_dtype and o.stride(1) == 1 and o.is_cuda, (o.shape, o.dtype)
            assert (o.stride(0) if M > 1 else ldo) == ldo and o.data_ptr() % 16 == 0, (o.stride(), ldo)
        ptrs = (ctypes.c_void_p * len(out_more))(*[o.data_ptr() for o in out_more])
        with _on_device(xq):
            rc = lib.pq_int8_gemm_bcast(xq.data_ptr(), ldx, s_row.data_ptr(), w_int8.data_ptr(), w_int8.stride(0),
                                        w_scale.data_ptr(), _ptr(bias), _ptr(t), ldt, _ptr(lb), ldb, _ptr(lb_t), R,
                                        _dt(out_dtype), out.data_ptr(), ptrs, len(out_more), _dt(out_dtype), ldo,
                                        M, N, K, int(epilogue), ws.data_ptr(), ws.numel() * 4, _stream(xq))
        if rc:
            _lib.check(rc, f"pq_int8_gemm_bcast(M={M}, N={N}, K={K}, copies={len(out_more)})")
        _written_in_place(out)
        for o in out_more:
            _written_in_place(o)
        return out
    if gate is not None:
        # out = out + gate[sample] * y (pq_int8_gemm_gated): gate [samples, N] in the output type; rows of sample b are
        # [b * gate_rows, (b + 1) * gate_rows)
        assert w_lo is None and dbg_acc is None and not out_more
        gate = gate.reshape(-1, N)
        assert gate.is_cuda and gate.dtype == out_dtype and gate.device == xq.device, (gate.dtype, out_dtype)
        assert gate.shape[0] == 1 or (gate_rows > 0 and gate.shape[0] * gate_rows >= M), (gate.shape, gate_rows, M)
        if gate.stride(1) != 1 or gate.stride(0) % 8 != 0 or gate.data_ptr() % 16 != 0:
            gate = gate.contiguous()
        assert epilogue_supported(N, ldo, out.data_ptr(), t is not None, R or 32), "shape needs the CTA-pair kernel"
        with _on_device(xq):
            rc = lib.pq_int8_gemm_gated(xq.data_ptr(), ldx, s_row.data_ptr(), w_int8.data_ptr(), w_int8.stride(0),
                                        w_scale.data_ptr(), _ptr(bias), _ptr(t), ldt, _ptr(lb), ldb, _ptr(lb_t), R,
                                        _dt(out_dtype), gate.data_ptr(), gate.stride(0) if gate.shape[0] > 1 else N,
                                        int(gate_rows) if gate.shape[0] > 1 else 0, out.data_ptr(), _dt(out_dtype), ldo,
                                        M, N, K, int(epilogue), ws.data_ptr(), ws.numel() * 4, _stream(xq))
        if rc:
            _lib.check(rc, f"pq_int8_gemm_gated(M={M}, N={N}, K={K})")
        _written_in_place(out)
        return out
    with _on_device(xq):
        if epilogue:
            assert w_lo is None and dbg_acc is None
            rc = lib.pq_int8_gemm_ex(xq.data_ptr(), ldx, s_row.data_ptr(), w_int8.data_ptr(), w_int8.stride(0),
                                     w_scale.data_ptr(), _ptr(bias), _ptr(t), ldt, _ptr(lb), ldb, _ptr(lb_t), R,
                                     _dt(out_dtype), out.data_ptr(), _dt(out_dtype), ldo,
                                     M, N, K, int(epilogue), ws.data_ptr(), ws.numel() * 4, _stream(xq))
        elif w_lo is None:
            rc = lib.pq_int8_gemm(xq.data_ptr(), ldx, s_row.data_ptr(), w_int8.data_ptr(), w_int8.stride(0),
                                  w_scale.data_ptr(), _ptr(bias), _ptr(t), ldt, _ptr(lb), ldb, _ptr(lb_t), R,
                                  _dt(out_dtype), out.data_ptr(), _dt(out_dtype), ldo, M, N, K, ws.data_ptr(), ws.numel() * 4,
                                  _ptr(dbg_acc), _stream(xq))
        else:
            assert w_lo.shape == w_int8.shape and w_lo.stride() == w_int8.stride() and s_lo is not None
            rc = lib.pq_int8_gemm_grouped(xq.data_ptr(), ldx, s_row.data_ptr(), w_int8.data_ptr(),
                                          w_scale.data_ptr(), w_lo.data_ptr(), s_lo.contiguous().data_ptr(),
                                          w_int8.stride(0), _ptr(bias), _ptr(t), ldt, _ptr(lb), ldb, _ptr(lb_t), R,
                                          _dt(out_dtype), out.data_ptr(), _dt(out_dtype), ldo, int(m_hi), M, N, K,
                                          ws.data_ptr(), ws.numel() * 4, _stream(xq))
    if rc:
        _lib.check(rc, f"pq_int8_gemm(M={M}, N={N}, K={K})")
    if epilogue & EPI_ACCUMULATE:
        _written_in_place(out)
    return out


def _gemm_g32_impl(xq: Tensor, s_a: Tensor, w_int8: Tensor, s_w_gm: Tensor, bias: Optional[Tensor],
                   out_dtype: torch.dtype) -> Tensor:
    """s_a [M, K/32]; s_w_gm [K/32, N] (group-major)."""
    assert xq.is_cuda and xq.dtype == torch.int8 and xq.dim() == 2 and w_int8.dtype == torch.int8
    M, K = xq.shape
    N = w_int8.shape[0]
    assert w_int8.shape[1] == K and K % 128 == 0, (w_int8.shape, K)
    assert s_a.shape == (M, K // 32) and s_w_gm.shape == (K // 32, N), (s_a.shape, s_w_gm.shape)
    assert bias is None or bias.numel() == N, f"bias has {bias.numel()} entries for {N} output channels"
    xq = xq.contiguous(); w_int8 = w_int8.contiguous()
    s_a = s_a.contiguous().float(); s_w_gm = s_w_gm.contiguous().float()
    if bias is not None:
        bias = bias.contiguous().float()
    out = torch.empty((M, N), dtype=out_dtype, device=xq.device)
    ws = status_word(xq.device)
    with _on_device(xq):
        rc = _LIB().pq_int8_gemm_g32(xq.data_ptr(), K, s_a.data_ptr(), w_int8.data_ptr(), K, s_w_gm.data_ptr(),
                                          _ptr(bias), out.data_ptr(), _dt(out_dtype), N, M, N, K, ws.data_ptr(),
                                          ws.numel() * 4, _stream(xq))
    _lib.check(rc, f"pq_int8_gemm_g32(M={M}, N={N}, K={K})")
    return out


def _dequant_epilogue_impl(acc: Tensor, s_row: Tensor, s_col: Tensor, bias: Optional[Tensor],
                           out_dtype: torch.dtype) -> Tensor:
    assert acc.is_cuda and acc.dtype == torch.int32 and acc.is_contiguous()
    M, N = acc.shape
    out = torch.empty((M, N), dtype=out_dtype, device=acc.device)
    with _on_device(acc):
        rc = _LIB().pq_dequant_epilogue(acc.data_ptr(), s_row.contiguous().data_ptr(),
                                             s_col.contiguous().data_ptr(), _ptr(bias), out.data_ptr(),
                                             _dt(out_dtype), M, N, _stream(acc))
    _lib.check(rc, "pq_dequant_epilogue")
    return out


def check_scatter_extents(m_act: int, canvas_rows: int, tokens: Tensor, ptr: Tensor, src: Tensor, beta: Tensor) -> None:
    """Extents of the contributor lists (their contents are trusted: they come from routing.build_route_plan)."""
    assert tokens.dim() == 1 and ptr.dim() == 1 and src.dim() == 1 and beta.dim() == 1
    assert ptr.numel() == tokens.numel() + 1, f"ptr has {ptr.numel()} entries for {tokens.numel()} tokens"
    assert src.numel() == beta.numel(), f"{src.numel()} sources but {beta.numel()} weights"
    assert tokens.numel() <= canvas_rows, f"{tokens.numel()} touched tokens on a canvas of {canvas_rows}"
    assert src.numel() == 0 or m_act > 0, "contributors without rows to take them from"


def _scatter_rows_impl(y: Tensor, tokens: Tensor, ptr: Tensor, src: Tensor, beta: Tensor, canvas: Tensor) -> None:
    assert y.is_cuda and canvas.is_cuda and y.dtype == canvas.dtype and y.dim() == 2 and canvas.dim() == 2
    assert y.stride(1) == 1 and canvas.stride(1) == 1 and y.shape[1] == canvas.shape[1]
    for v in (tokens, ptr, src):
        assert v.is_cuda and v.dtype == torch.int32 and v.is_contiguous()
    assert beta.is_cuda and beta.dtype == torch.float32 and beta.is_contiguous()
    n_tokens = tokens.numel()
    check_scatter_extents(y.shape[0], canvas.shape[0], tokens, ptr, src, beta)
    with _on_device(canvas):
        rc = _LIB().pq_scatter_rows(y.data_ptr(), max(y.stride(0), y.shape[1]), y.shape[0], tokens.data_ptr(),
                                         ptr.data_ptr(), src.data_ptr(), beta.data_ptr(), n_tokens,
                                         canvas.data_ptr(), max(canvas.stride(0), canvas.shape[1]), canvas.shape[0],
                                         canvas.shape[1], _dt(canvas.dtype), _stream(canvas))
    _lib.check(rc, "pq_scatter_rows")


def fuse_rows(background: Tensor, y: Tensor, tokens: Tensor, ptr: Tensor, src: Tensor, beta: Tensor, rest: Tensor) -> Tensor:
    """A new [rows, C] tensor: the routed rows blended over `background` at `tokens`, the background's rows at `rest`
    (pq_fuse_rows)."""
    assert y.is_cuda and background.is_cuda and y.dtype == background.dtype and y.dim() == 2 and background.dim() == 2
    assert y.stride(1) == 1 and background.stride(1) == 1 and y.shape[1] == background.shape[1]
    for v in (tokens, ptr, src, rest):
        assert v.is_cuda and v.dtype == torch.int32 and v.is_contiguous()
    assert beta.is_cuda and beta.dtype == torch.float32 and beta.is_contiguous()
    rows, C = background.shape
    check_scatter_extents(y.shape[0], rows, tokens, ptr, src, beta)
    assert tokens.numel() + rest.numel() == rows, (tokens.numel(), rest.numel(), rows)
    out = torch.empty((rows, C), dtype=y.dtype, device=background.device)
    with _on_device(background):
        rc = _LIB().pq_fuse_rows(y.data_ptr(), max(y.stride(0), C), y.shape[0], tokens.data_ptr(), ptr.data_ptr(), src.data_ptr(),
                                 beta.data_ptr(), tokens.numel(), rest.data_ptr(), rest.numel(), background.data_ptr(),
                                 max(background.stride(0), C), out.data_ptr(), C, rows, C, _dt(y.dtype), _stream(background))
    _lib.check(rc, "pq_fuse_rows")
    return out


# ------------------------------------------------------------------------------------------------ custom ops
# torch.library schemas cannot carry torch.dtype arguments portably, so out_dtype travels as the dtype code.
_CODE2DT = {_lib.DTYPE_BF16: torch.bfloat16, _lib.DTYPE_FP16: torch.float16}


@torch.library.custom_op("pq_b200::quant_rows", mutates_args=(), device_types="cuda")
def quant_rows_op(x2: Tensor) -> Tuple[Tensor, Tensor]:
    return _quant_rows_impl(x2)


@quant_rows_op.register_fake
def _(x2):
    return x2.new_empty(x2.shape, dtype=torch.int8), x2.new_empty((x2.shape[0],), dtype=torch.float32)


@torch.library.custom_op("pq_b200::quant_rows_g32", mutates_args=(), device_types="cuda")
def quant_rows_g32_op(x2: Tensor) -> Tuple[Tensor, Tensor]:
    return _quant_rows_g32_impl(x2)


@quant_rows_g32_op.register_fake
def _(x2):
    return (x2.new_empty(x2.shape, dtype=torch.int8),
            x2.new_empty((x2.shape[0], x2.shape[1] // 32), dtype=torch.float32))


@torch.library.custom_op("pq_b200::gather_quant_rows", mutates_args=(), device_types="cuda")
def gather_quant_rows_op(canvas: Tensor, row_idx: Tensor) -> Tuple[Tensor, Tensor]:
    return _gather_quant_rows_impl(canvas, row_idx)


@gather_quant_rows_op.register_fake
def _(canvas, row_idx):
    M = row_idx.shape[0]
    return canvas.new_empty((M, canvas.shape[1]), dtype=torch.int8), canvas.new_empty((M,), dtype=torch.float32)


@torch.library.custom_op("pq_b200::gather_rows", mutates_args=(), device_types="cuda")
def gather_rows_op(canvas: Tensor, row_idx: Tensor) -> Tensor:
    return _gather_rows_impl(canvas, row_idx)


@gather_rows_op.register_fake
def _(canvas, row_idx):
    return canvas.new_empty((row_idx.shape[0], canvas.shape[1]))


@torch.library.custom_op("pq_b200::int8_gemm", mutates_args=(), device_types="cuda")
def int8_gemm_op(xq: Tensor, s_row: Tensor, w_int8: Tensor, w_scale: Tensor, bias: Optional[Tensor],
                 t: Optional[Tensor], lb: Optional[Tensor], out_dtype_code: int,
                 lb_t: Optional[Tensor] = None) -> Tensor:
    return _gemm_impl(xq, s_row, w_int8, w_scale, bias, t, lb, _CODE2DT[out_dtype_code], lb_t=lb_t)


@int8_gemm_op.register_fake
def _(xq, s_row, w_int8, w_scale, bias, t, lb, out_dtype_code, lb_t=None):
    return xq.new_empty((xq.shape[0], w_int8.shape[0]), dtype=_CODE2DT[out_dtype_code])


@torch.library.custom_op("pq_b200::int8_gemm_grouped", mutates_args=(), device_types="cuda")
def int8_gemm_grouped_op(xq: Tensor, s_row: Tensor, w_hi: Tensor, s_hi: Tensor, w_lo: Tensor, s_lo: Tensor,
                         bias: Optional[Tensor], t: Optional[Tensor], lb: Optional[Tensor], m_hi: int,
                         out_dtype_code: int, lb_t: Optional[Tensor] = None) -> Tensor:
    return _gemm_impl(xq, s_row, w_hi, s_hi, bias, t, lb, _CODE2DT[out_dtype_code], None, w_lo, s_lo, m_hi, lb_t)


@int8_gemm_grouped_op.register_fake
def _(xq, s_row, w_hi, s_hi, w_lo, s_lo, bias, t, lb, m_hi, out_dtype_code, lb_t=None):
    return xq.new_empty((xq.shape[0], w_hi.shape[0]), dtype=_CODE2DT[out_dtype_code])


@torch.library.custom_op("pq_b200::int8_gemm_g32", mutates_args=(), device_types="cuda")
def int8_gemm_g32_op(xq: Tensor, s_a: Tensor, w_int8: Tensor, s_w_gm: Tensor, bias: Optional[Tensor],
                     out_dtype_code: int) -> Tensor:
    return _gemm_g32_impl(xq, s_a, w_int8, s_w_gm, bias, _CODE2DT[out_dtype_code])


@int8_gemm_g32_op.register_fake
def _(xq, s_a, w_int8, s_w_gm, bias, out_dtype_code):
    return xq.new_empty((xq.shape[0], w_int8.shape[0]), dtype=_CODE2DT[out_dtype_code])


def _fp4_lowrank_rows_impl(t: Tensor, row_scale: Optional[Tensor]) -> Tensor:
    out = _BIND().fp4_lowrank_rows(t, row_scale)
    if out is not None:
        return out
    dt = _dt(t.dtype)
    assert t.is_cuda and t.dim() == 2 and t.shape[1] == 32, "low-rank activations are [M, 32] on a GPU"
    M = t.shape[0]
    assert row_scale is None or (row_scale.dtype == torch.float32 and row_scale.numel() == M and row_scale.is_contiguous()
                                 and row_scale.device == t.device), "one fp32 row scale per row"
    if not t.is_contiguous() or t.data_ptr() % 16 != 0:
        t = t.clone(memory_format=torch.contiguous_format)
    out = t.new_empty((M, 32), dtype=torch.float32)
    with _on_device(t):
        rc = _LIB().pq_fp4_lowrank_rows(t.data_ptr(), dt, _ptr(row_scale), out.data_ptr(), M, _stream(t))
    if rc:
        _lib.check(rc, f"pq_fp4_lowrank_rows(M={M})")
    return out


def _fp4_lowrank_factors_impl(t: Tensor, row_scale: Optional[Tensor], B: Tensor, col_scale: Optional[Tensor]) -> Tuple[Tensor, Tensor]:
    out = _BIND().fp4_lowrank_factors(t, row_scale, B, col_scale)
    if out is not None:
        return out
    dt, db = _dt(t.dtype), _dt(B.dtype)
    assert t.is_cuda and t.dim() == 2 and t.shape[1] == 32, "low-rank activations are [M, 32] on a GPU"
    assert B.dim() == 2 and B.shape[0] == 32 and B.device == t.device, "the up-projection is [32, N] on the activations' device"
    M, N = t.shape[0], B.shape[1]
    for s, n in ((row_scale, M), (col_scale, N)):
        assert s is None or (s.dtype == torch.float32 and s.numel() == n and s.is_contiguous() and s.device == t.device), \
            "one fp32 row scale per row"
    if not t.is_contiguous() or t.data_ptr() % 16 != 0:
        t = t.clone(memory_format=torch.contiguous_format)
    if not B.is_contiguous():
        B = B.contiguous()
    t_out, b_out = t.new_empty((M, 32), dtype=torch.float32), t.new_empty((N, 32), dtype=torch.float32)
    with _on_device(t):
        rc = _LIB().pq_fp4_lowrank_factors(t.data_ptr(), dt, _ptr(row_scale), t_out.data_ptr(), M, B.data_ptr(), db, N, _ptr(col_scale),
                                           b_out.data_ptr(), N, _stream(t))
    if rc:
        _lib.check(rc, f"pq_fp4_lowrank_factors(M={M}, N={N})")
    return t_out, b_out


@torch.library.custom_op("pq_b200::group_norm_rows", mutates_args=(), device_types="cuda")
def group_norm_rows_op(x: Tensor, groups: int, weight: Optional[Tensor], bias: Optional[Tensor], eps: float, silu: bool) -> Tensor:
    return _group_norm_impl(x, groups, weight, bias, eps, "silu" if silu else None)


@group_norm_rows_op.register_fake
def _(x, groups, weight, bias, eps, silu):
    return x.new_empty(x.shape)


# 4-bit rows travel as (codes, scales, row scales); an operator cannot return an optional tensor, so the mx format's absent
# row scales are an empty tensor here.
@torch.library.custom_op("pq_b200::quant_rows_fp4", mutates_args=(), device_types="cuda")
def quant_rows_fp4_op(x2: Tensor, fmt: str) -> Tuple[Tensor, Tensor, Tensor]:
    codes, scales, row = _quant_rows_fp4_impl(x2, fmt)
    return codes, scales, row if row is not None else scales.new_empty((0,), dtype=torch.float32)


@quant_rows_fp4_op.register_fake
def _(x2, fmt):
    M, K = x2.shape
    return (x2.new_empty((M, K // 2), dtype=torch.uint8), x2.new_empty(fp4_scale_shape(M, K, fmt), dtype=torch.uint8),
            x2.new_empty((M if fmt == "nv" else 0,), dtype=torch.float32))


@torch.library.custom_op("pq_b200::dequant_rows_fp4", mutates_args=(), device_types="cuda")
def dequant_rows_fp4_op(codes: Tensor, scales: Tensor, row_scale: Optional[Tensor], dtype_code: int) -> Tensor:
    return _dequant_rows_fp4_impl(codes, scales, row_scale, _CODE2DT[dtype_code])


@dequant_rows_fp4_op.register_fake
def _(codes, scales, row_scale, dtype_code):
    return codes.new_empty((codes.shape[0], codes.shape[1] * 2), dtype=_CODE2DT[dtype_code])


@torch.library.custom_op("pq_b200::fp4_gemm", mutates_args=(), device_types="cuda")
def fp4_gemm_op(xq: Tensor, xs: Tensor, x_row: Optional[Tensor], wq: Tensor, ws: Tensor, w_row: Optional[Tensor],
                bias: Optional[Tensor], out_dtype_code: int, t: Optional[Tensor] = None, lb: Optional[Tensor] = None) -> Tensor:
    return _fp4_gemm_impl(xq, xs, x_row, wq, ws, w_row, bias, _CODE2DT[out_dtype_code], t, lb)


@fp4_gemm_op.register_fake
def _(xq, xs, x_row, wq, ws, w_row, bias, out_dtype_code, t=None, lb=None):
    return xq.new_empty((xq.shape[0], wq.shape[0]), dtype=_CODE2DT[out_dtype_code])


@torch.library.custom_op("pq_b200::fp4_lowrank_rows", mutates_args=(), device_types="cuda")
def fp4_lowrank_rows_op(t: Tensor, row_scale: Optional[Tensor]) -> Tensor:
    return _fp4_lowrank_rows_impl(t, row_scale)


@fp4_lowrank_rows_op.register_fake
def _(t, row_scale):
    return t.new_empty((t.shape[0], 32), dtype=torch.float32)


@torch.library.custom_op("pq_b200::dequant_epilogue", mutates_args=(), device_types="cuda")
def dequant_epilogue_op(acc: Tensor, s_row: Tensor, s_col: Tensor, bias: Optional[Tensor],
                        out_dtype_code: int) -> Tensor:
    return _dequant_epilogue_impl(acc, s_row, s_col, bias, _CODE2DT[out_dtype_code])


@dequant_epilogue_op.register_fake
def _(acc, s_row, s_col, bias, out_dtype_code):
    return acc.new_empty(acc.shape, dtype=_CODE2DT[out_dtype_code])


@torch.library.custom_op("pq_b200::scatter_rows_", mutates_args=("canvas",), device_types="cuda")
def scatter_rows_op(y: Tensor, tokens: Tensor, ptr: Tensor, src: Tensor, beta: Tensor, canvas: Tensor) -> None:
    _scatter_rows_impl(y, tokens, ptr, src, beta, canvas)


def dtype_code(dtype: torch.dtype) -> int:
    return _dt(dtype)


def int8_gemm_debug(xq: Tensor, s_row: Tensor, w_int8: Tensor, w_scale: Tensor, bias: Optional[Tensor],
                    t: Optional[Tensor], lb: Optional[Tensor], out_dtype: torch.dtype) -> Tuple[Tensor, Tensor]:
    """GEMM that also returns the raw int32 accumulators (parity tests)."""
    acc = torch.full((xq.shape[0], w_int8.shape[0]), -2**31, dtype=torch.int32, device=xq.device)
    out = _gemm_impl(xq, s_row, w_int8, w_scale, bias, t, lb, out_dtype, dbg_acc=acc)
    return out, acc
