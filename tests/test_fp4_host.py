"""4-bit floating-point Linears, host side: weight quantisation against the 64-bit restatement, module and conversion logic,
and the argument checks of the C ABI (no GPU needed)."""
import ctypes

import pytest
import torch
import torch.nn as nn

from oracle import fp4 as ofp4
from pyraquant_b200 import _lib, fp4_exec, ops

FMTS = ["mx", "nv"]


def awkward_rows(M, K, dtype, seed):
    """Rows over a wide range of magnitudes, with zeros, zero blocks, and values on the borders between codes."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(M, K, generator=g) * torch.exp2(torch.randint(-6, 7, (M, 1), generator=g).float())
    x[:, torch.randperm(K, generator=g)[: max(1, K // 100)]] *= 30
    x[torch.rand(M, K, generator=g) < 0.02] = 0
    if M > 4:
        x[1] = 0
        x[2, : K // 2] = 0
        x[3] = torch.tensor([6, 0.25, -0.75, 1.25, -1.75, 2.5, -3.5, 5, -0.25, 0.75, -5, 0.5, 3, -0.0, 4, 1.0]).repeat(K // 16) * 2.0 ** -3
        x[4] = x[3] * 1.5
    return x.to(dtype)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("N,K", [(1, 32), (5, 64), (130, 96), (257, 640)])
def test_weight_quantisation_matches_the_definition(fmt, dtype, N, K):
    w = awkward_rows(N, K, dtype, N + K)
    q = fp4_exec.quantize_weight_fp4(w, fmt)
    code, byte, row = ofp4.quantise(w, fmt)
    assert q.fmt == fmt and q.codes.shape == (N, K // 2) and tuple(q.scales.shape) == ops.fp4_scale_shape(N, K, fmt)
    assert torch.equal(ofp4.untile(q.scales, N, K, fmt), byte)
    assert (q.row_scale is None) == (row is None) and (row is None or torch.equal(q.row_scale.double(), row))
    # the sign of a zero is free where the block's scale is zero
    got, want = ofp4.unpack(q.codes), code
    assert torch.equal(got % 8, want % 8)
    nz = want % 8 != 0
    assert torch.equal(got[nz], want[nz])
    assert int(q.scales.sum()) == int(byte.sum())                 # nothing outside the rows and blocks


@pytest.mark.parametrize("fmt", FMTS)
def test_quantised_values_are_near(fmt):
    """Every value is within half the local step of E2M1 of the original, short of the clipped top of an mx block."""
    x = awkward_rows(64, 256, torch.bfloat16, 9)
    code, byte, row = ofp4.quantise(x, fmt)
    v = ofp4.values(code, byte, row, fmt)
    s = (v.new_tensor(2.0) ** (byte.double() - 127) if fmt == "mx" else ofp4.E4M3[byte] * row[:, None]).repeat_interleave(ofp4.BLOCK[fmt], 1)
    a = x.double().abs() / s.clamp_min(1e-300)
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    inside = (a <= 6) & (s > 0)
    assert bool(((v - x.double()).abs()[inside] <= (step * s)[inside] / 2).all())
    if fmt == "mx":
        assert float(a.max()) < 8                                # the top of a block is clipped from below 8 to 6


def test_modules_and_conversion():
    torch.manual_seed(0)
    lin = nn.Linear(64, 40)
    for fmt in FMTS:
        m = fp4_exec.Fp4Linear(lin, fmt=fmt)
        assert m.weight_rows.fmt == fmt and m.bias.dtype == torch.float32 and m.lr_A is None
        again = fp4_exec.Fp4Linear(nn.Linear(64, 40), fmt=fmt)
        again.load_state_dict(m.state_dict())
        assert all(torch.equal(a, b) for a, b in zip(again.state_dict().values(), m.state_dict().values()))
        before = {k: v.clone() for k, v in m.state_dict().items()}
        m.half()
        assert all(torch.equal(v, before[k]) and v.dtype == before[k].dtype for k, v in m.state_dict().items())
        with pytest.raises(AssertionError):
            m(torch.randn(3, 64))                                # CPU tensors are refused
    net = nn.ModuleDict({"a": nn.Linear(64, 32), "b": nn.Linear(48, 32), "proj_out": nn.Linear(64, 64)})
    st = fp4_exec.convert_linears_to_fp4(net, device=None, fmt="mx")
    assert isinstance(net["a"], fp4_exec.Fp4Linear) and st["n_fp4_linear"] == 1 and st["params_fp4"] == 64 * 32
    assert sorted(st["bf16_kept_names"]) == ["b", "proj_out"]      # 48 is no multiple of 32, proj_out is kept by name


def test_refusals():
    with pytest.raises(ValueError):
        fp4_exec.quantize_weight_fp4(torch.randn(4, 64), "e5")
    with pytest.raises(AssertionError):
        fp4_exec.quantize_weight_fp4(torch.randn(4, 48), "mx")
    with pytest.raises(AssertionError):
        fp4_exec.quantize_weight_fp4(torch.full((4, 64), float("inf")), "nv")
    for call in (lambda: fp4_exec.quant_rows_fp4(torch.randn(4, 64, dtype=torch.bfloat16)),
                 lambda: fp4_exec.dequant_rows_fp4(fp4_exec.quantize_weight_fp4(torch.randn(4, 64))),
                 lambda: fp4_exec.fp4_gemm(fp4_exec.quantize_weight_fp4(torch.randn(4, 64)), fp4_exec.quantize_weight_fp4(torch.randn(4, 64)))):
        with pytest.raises(AssertionError):
            call()                                               # CPU tensors


def test_one_step_calls_leave_other_operands_to_the_general_path():
    """The one-step calls answer None, without touching anything, for what they do not take as it is."""
    bind = _lib.binding()
    x = torch.randn(4, 64, dtype=torch.bfloat16)
    q = fp4_exec.quantize_weight_fp4(x)
    assert bind.quant_rows_fp4(x, 1) is None and bind.quant_rows_fp4(None, 1) is None and bind.quant_rows_fp4(3, 1) is None
    assert bind.dequant_rows_fp4(*q, True) is None and bind.dequant_rows_fp4(q.codes, 5, None, True) is None
    assert bind.fp4_gemm(*q, *q, None, True, 0, 0) is None and bind.fp4_gemm(*q, *q, "bias", True, 0, 0) is None
    assert bind.fp4_gemm(*q, *q, None, True, 0, 0, None, None) is None and bind.fp4_gemm(*q, *q, None, True, 0, 0, x, None) is None
    assert bind.fp4_gemm(*q, *q, None, True, 0, 0, "t", 3) is None
    assert bind.fp4_lowrank_rows(x[:, :32], None) is None and bind.fp4_lowrank_rows("t", None) is None and bind.fp4_lowrank_rows(x) is None
    assert bind.group_norm(x[None], 4, None, None, 1e-6, 0, 0, True, 0) is None
    assert bind.group_norm(x[None], 4.0, "w", None, 1e-6, 0, 0, True, 0) is None


def test_argument_checks():
    lib = _lib.load()
    buf = ctypes.create_string_buffer(8192)
    p = (ctypes.addressof(buf) + 63) & ~63
    NULL, SHAPE, ALIGN, DTYPE, UNSUPPORTED, WORKSPACE = 1, 2, 3, 4, 7, 8

    assert lib.pq_fp4_scale_bytes(1, 32, 0) == 512 and lib.pq_fp4_scale_bytes(129, 160, 0) == 2 * 2 * 512
    assert lib.pq_fp4_scale_bytes(128, 160, 1) == 3 * 512 and lib.pq_fp4_scale_bytes(0, 64, 1) == 0
    assert lib.pq_fp4_scale_bytes(-1, 64, 0) == 0 and lib.pq_fp4_scale_bytes(1, 64, 2) == 0

    def quant(x=p, dtype=0, M=4, K=64, ldx=64, fmt=1, codes=p, scales=p, row=p):
        return lib.pq_quant_rows_fp4(x, dtype, M, K, ldx, fmt, codes, scales, row, None)
    assert quant(M=0, x=None) == 0
    assert quant(x=None) == NULL and quant(codes=None) == NULL and quant(scales=None) == NULL and quant(row=None) == NULL
    assert quant(dtype=3) == DTYPE and quant(fmt=5) == UNSUPPORTED
    assert quant(M=-1) == SHAPE and quant(K=0) == SHAPE and quant(ldx=32) == SHAPE
    assert quant(K=48, ldx=48) == ALIGN and quant(ldx=72) == ALIGN and quant(x=p + 16) == ALIGN and quant(codes=p + 8) == ALIGN

    def dequant(codes=p, ldc=32, scales=p, row=p, fmt=1, out=p, dtype=0, ldo=64, M=4, K=64):
        return lib.pq_dequant_rows_fp4(codes, ldc, scales, row, fmt, out, dtype, ldo, M, K, None)
    assert dequant(M=0, codes=None) == 0
    assert dequant(codes=None) == NULL and dequant(row=None) == NULL and dequant(out=None) == NULL
    assert dequant(ldc=16) == SHAPE and dequant(ldo=32) == SHAPE and dequant(dtype=9) == DTYPE and dequant(fmt=-1) == UNSUPPORTED
    assert dequant(ldc=40) == ALIGN and dequant(out=p + 16) == ALIGN and dequant(ldo=72) == ALIGN

    def gemm(xq=p, ldx=32, xs=p, sr=p, w=p, ldw=32, wsc=p, sc=p, bias=None, fmt=1, out=p, dtype=0, ldo=40, M=4, N=40, K=64,
             ws=None, wsb=0):
        return lib.pq_fp4_gemm(xq, ldx, xs, sr, w, ldw, wsc, sc, bias, fmt, out, dtype, ldo, M, N, K, ws, wsb, None)
    assert gemm(M=0, xq=None) == 0
    for name in ("xq", "xs", "w", "wsc", "out", "sr", "sc"):
        assert gemm(**{name: None}) == NULL, name
    assert gemm(N=0) == SHAPE and gemm(ldx=16) == SHAPE and gemm(ldw=16) == SHAPE and gemm(ldo=39) == SHAPE
    assert gemm(K=48, ldx=32, ldw=32) == ALIGN and gemm(ldx=40) == ALIGN and gemm(w=p + 8) == ALIGN and gemm(out=p + 1) == ALIGN
    assert gemm(dtype=2) == DTYPE and gemm(fmt=3) == UNSUPPORTED and gemm(ws=p, wsb=8) == WORKSPACE

    def low(t=p, lb=p, M=4, K=64, fmt=1, sr=p):
        return lib.pq_fp4_gemm_lowrank(p, 32, p, sr, p, 32, p, p, None, t, lb, fmt, p, 0, 40, M, 40, K, None, 0, None)
    assert low(M=0) == 0 and low(t=None) == NULL and low(lb=None) == NULL and low(sr=None) == NULL
    assert low(t=p + 8) == ALIGN and low(lb=p + 4) == ALIGN and low(K=0) == SHAPE and low(fmt=2) == UNSUPPORTED

    def rows(t=p, dtype=0, row=p, out=p, M=4):
        return lib.pq_fp4_lowrank_rows(t, dtype, row, out, M, None)
    assert rows(M=0, t=None) == 0 and rows(t=None) == NULL and rows(out=None) == NULL and rows(M=-1) == SHAPE and rows(dtype=2) == DTYPE
    assert rows(t=p + 8) == ALIGN and rows(out=p + 16) == ALIGN and rows(row=p + 2) == ALIGN
