"""4-bit floating-point operators on the GPU against the 64-bit restatement: codes, scales and values bit for bit, products
within a bound derived from the formats' arithmetic.

Bound of a product.  Every product of two values is exact in fp32 (at most 2 x 2 significant bits times scales of 2 x 4).
One MMA adds 64 of them to the fp32 accumulator; with S = sum |x w| over the row of K, aligning and adding inside an MMA
loses at most 2 units of 2^-23 S and so does adding its sum to the accumulator: 4 * 2^-23 S per 64 elements, K / 16 * 2^-23 S
in all.  Joining up to eight partial sums of a split launch: 8 * 2^-24 S.  Row scales are powers of two (exact); the bias
adds once more (2^-24 of the sum's size).  The rounding to 16 bits is half a step: eps / 2 of the value, or half the
smallest subnormal.
"""
import pytest
import torch
import torch.nn as nn

from oracle import fp4 as ofp4
from pyraquant_b200 import _lib, fp4_exec, ops
from test_fp4_host import awkward_rows

pytestmark = pytest.mark.gpu
FMTS = ["mx", "nv"]
DTYPES = [torch.bfloat16, torch.float16]


@pytest.fixture(autouse=True)
def _status_clean(cuda_dev):
    yield
    _lib.set_option("fp4_pair", 1)
    _lib.set_option("fp4_split", 0)
    ops.check_device_status(cuda_dev)


def check_rows(q, x, fmt):
    code, byte, row = ofp4.quantise(x.cpu(), fmt)
    M, K = x.shape
    assert q.fmt == fmt and torch.equal(ofp4.untile(q.scales.cpu(), M, K, fmt), byte)
    if fmt == "nv":
        assert torch.equal(q.row_scale.cpu().double(), row)
    got = ofp4.unpack(q.codes.cpu())
    assert torch.equal(got % 8, code % 8)
    nz = code % 8 != 0
    assert torch.equal(got[nz], code[nz])


def check_product(y, xq, wq, bias, fmt):
    """y against the 64-bit product of the packed rows."""
    X = ofp4.packed_values(xq.codes.cpu(), xq.scales.cpu(), None if xq.row_scale is None else xq.row_scale.cpu(), fmt)
    W = ofp4.packed_values(wq.codes.cpu(), wq.scales.cpu(), None if wq.row_scale is None else wq.row_scale.cpu(), fmt)
    K = X.shape[1]
    ref = X @ W.t()
    S = X.abs() @ W.abs().t()
    bound = (K / 16 + 4) * 2.0 ** -23 * S
    if bias is not None:
        ref = ref + bias.cpu().double()
        bound = bound + 2.0 ** -24 * (S + bias.cpu().double().abs())
    fi = torch.finfo(y.dtype)
    bound = bound + (ref.abs() + bound) * fi.eps / 2 + fi.smallest_normal * fi.eps / 2
    got = y.cpu().double()
    # 16-bit rounding: from half a step above the largest finite value on, an infinity of the sum's sign
    border = fi.max * (2 - fi.eps / 2) / (2 - fi.eps)
    beyond, inside = ref.abs() - bound >= border, ref.abs() + bound < border
    assert torch.equal(got[beyond], torch.sign(ref[beyond]) * float("inf")) and bool(torch.isfinite(got[inside]).all())
    err = torch.where(inside, (got - ref).abs(), torch.zeros_like(ref))
    worst = float((err / bound).max())
    assert worst <= 1, f"error {worst:.3g} times the bound at {divmod(int((err / bound).argmax()), y.shape[1])}"


def make_rows(M, K, fmt, dtype, seed, dev):
    x = awkward_rows(M, K, dtype, seed).to(dev)
    return x, fp4_exec.quant_rows_fp4(x, fmt)


# ------------------------------------------------------------------------------------------------ quantisation
@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,K", [(1, 32), (3, 64), (33, 96), (127, 640), (129, 672), (300, 1280), (70, 2560), (65, 2592), (40, 5120),
                                 (9, 10240), (5, 12288), (7, 20480), (3, 20512), (2, 40960)])
def test_quant_rows_match_the_definition(cuda_dev, fmt, dtype, M, K):
    x = awkward_rows(M, K, dtype, M * 7 + K)
    check_rows(fp4_exec.quant_rows_fp4(x.to(cuda_dev), fmt), x, fmt)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("dtype", DTYPES)
def test_quant_every_significand_against_every_block_maximum(cuda_dev, fmt, dtype):
    """Blocks whose maximum runs over every significand of the type and whose other elements run over the binades below:
    every border between codes that the type can hit, exactly and from both sides."""
    one, per, step = (0x3F80, 128, 1) if dtype == torch.bfloat16 else (0x3C00, 1024, 8)
    n = 16 if fmt == "nv" else 32
    amax = torch.arange(one, one + per, step, dtype=torch.int32)
    below = torch.arange(0, 5 * per, step, dtype=torch.int32)
    below = torch.nn.functional.pad(below, (0, (-below.numel()) % (n - 1)))
    rest = (amax[:, None] - below[None, :]).reshape(amax.numel(), -1, n - 1)
    bits = torch.cat([amax[:, None, None].expand(-1, rest.shape[1], 1), rest], dim=2).reshape(amax.numel(), -1)
    bits = torch.nn.functional.pad(bits, (0, (-bits.shape[1]) % 32))
    bits[:, 1::2] |= 0x8000
    x = torch.where(bits >= 0x8000, bits - 0x10000, bits).to(torch.int16).view(dtype)
    check_rows(fp4_exec.quant_rows_fp4(x.to(cuda_dev), fmt), x, fmt)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("dtype", DTYPES)
def test_quant_keeps_the_sign_of_zeros(cuda_dev, dtype, fmt):
    """Every byte is that of the plain arithmetic, the signs of zeros and of what rounds to zero among them."""
    x = awkward_rows(64, 640, dtype, 9).float()
    g = torch.Generator().manual_seed(10)
    pick = torch.rand(x.shape, generator=g)
    x = torch.where(pick < 0.2, torch.full_like(x, -0.0), torch.where(pick < 0.3, torch.zeros_like(x), torch.where(pick < 0.4, x * 1e-3, x)))
    x[5] = -0.0
    x = x.to(dtype).to(cuda_dev)
    got, want = fp4_exec.quant_rows_fp4(x, fmt), fp4_exec.quantize_weight_fp4(x, fmt)
    assert torch.equal(got.codes, want.codes)
    kept = (got.codes & 8 != 0) == torch.signbit(x[:, 0::2])                          # wherever the block's scale is not zero
    zero_scale = (fp4_exec.dequant_rows_fp4(want) == 0).reshape(64, -1, ops.FP4_BLOCK[fmt]).all(2).repeat_interleave(ops.FP4_BLOCK[fmt], 1)
    assert bool((kept | zero_scale[:, 0::2]).all())


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("dtype", DTYPES)
def test_quant_every_magnitude(cuda_dev, fmt, dtype):
    """Every positive finite value of the type as the maximum of a row: row scales, block scales and codes over the whole
    exponent range, subnormals among them."""
    top = 0x7F80 if dtype == torch.bfloat16 else 0x7C00
    v = torch.arange(1, top, dtype=torch.int32).to(torch.int16).view(dtype)
    x = torch.stack([v * f for f in (1.0, 0.75, -0.4, 0.1)], dim=1).repeat(1, 8)
    check_rows(fp4_exec.quant_rows_fp4(x.to(cuda_dev), fmt), x, fmt)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("dtype", DTYPES)
def test_read_back(cuda_dev, fmt, dtype):
    for M, K in ((1, 32), (130, 672), (37, 5120)):
        x, q = make_rows(M, K, fmt, dtype, M + K, cuda_dev)
        want = ofp4.packed_values(q.codes.cpu(), q.scales.cpu(), None if q.row_scale is None else q.row_scale.cpu(), fmt)
        for t in DTYPES:
            w = want.clamp(-65504, 65504) if t == torch.float16 else want
            assert torch.equal(fp4_exec.dequant_rows_fp4(q, t).cpu(), w.to(t))
    big = torch.full((1, 32), 65504.0, dtype=torch.float16, device=cuda_dev)
    assert torch.isfinite(fp4_exec.dequant_rows_fp4(fp4_exec.quant_rows_fp4(big, fmt), torch.float16)).all()


@pytest.mark.parametrize("fmt", FMTS)
def test_infinities_and_nan(cuda_dev, fmt):
    x = torch.randn(6, 96, generator=torch.Generator().manual_seed(3)).to(torch.bfloat16)
    x[1, 40] = float("inf"); x[3, 0] = float("nan"); x[4, 95] = float("-inf")
    q = fp4_exec.quant_rows_fp4(x.to(cuda_dev), fmt)
    v = fp4_exec.dequant_rows_fp4(q, torch.bfloat16).cpu()
    bad = torch.zeros(6, 96, dtype=torch.bool)
    if fmt == "mx":
        bad[1, 32:64] = True; bad[3, :32] = True; bad[4, 64:] = True
    else:
        bad[[1, 3, 4]] = True
    assert torch.equal(torch.isnan(v), bad)
    clean = torch.where(bad, torch.zeros_like(x), x)
    good = ofp4.values(*ofp4.quantise(clean, fmt), fmt).to(torch.bfloat16)
    assert torch.equal(v[~bad], good[~bad])
    w = fp4_exec.quantize_weight_fp4(torch.randn(40, 96, generator=torch.Generator().manual_seed(4)), fmt)
    w = fp4_exec.Fp4Rows(*(None if t is None else t.to(cuda_dev) for t in w))
    y = fp4_exec.fp4_gemm(q, w, None, torch.bfloat16).cpu()
    assert torch.isnan(y[[1, 3, 4]]).all() and torch.isfinite(y[[0, 2, 5]]).all()


def test_quant_strided_and_offset_rows(cuda_dev):
    x = awkward_rows(50, 1280, torch.bfloat16, 5).to(cuda_dev)
    for fmt in FMTS:
        for view in (x[:, 640:], x[::2], x[3:, :64], x[:, 8:648], x.t()[:32].t(), x[:, ::2], x[7:8, 16:48]):
            check_rows(fp4_exec.quant_rows_fp4(view, fmt), view, fmt)
        empty = fp4_exec.quant_rows_fp4(x[:0], fmt)
        assert empty.codes.shape == (0, 640) and empty.scales.shape[0] == 0


# ------------------------------------------------------------------------------------------------ product
@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("M,N,K", [(128, 64, 256), (1, 64, 32), (1, 1, 64), (5, 7, 96), (128, 128, 64), (77, 200, 640), (16, 1288, 160),
                                   (200, 72, 2592), (129, 130, 288), (1, 1280, 5120), (33, 650, 2048)])
def test_product(cuda_dev, fmt, M, N, K):
    dtype = DTYPES[(M + N) % 2]
    _, xq = make_rows(M, K, fmt, dtype, 1, cuda_dev)
    _, wq = make_rows(N, K, fmt, torch.bfloat16, 2, cuda_dev)
    bias = torch.randn(N, device=cuda_dev) if N % 2 else None
    check_product(fp4_exec.fp4_gemm(xq, wq, bias, torch.bfloat16), xq, wq, bias, fmt)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("M,N,K", [(2048, 2176, 640), (2500, 1990, 480), (4173, 640, 2560)])
def test_product_many_tiles(cuda_dev, fmt, M, N, K):
    g = torch.Generator().manual_seed(6)
    x = torch.randn(M, K, generator=g).to(torch.float16).to(cuda_dev)
    w = torch.randn(N, K, generator=g).to(torch.bfloat16).to(cuda_dev)
    xq, wq = fp4_exec.quant_rows_fp4(x, fmt), fp4_exec.quant_rows_fp4(w, fmt)
    bias = torch.randn(N, generator=g).to(cuda_dev)
    check_product(fp4_exec.fp4_gemm(xq, wq, bias, torch.bfloat16), xq, wq, bias, fmt)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("split", [1, 2, 4, 8])
@pytest.mark.parametrize("M,N,K", [(1, 640, 2560), (77, 200, 2080), (130, 70, 5120), (300, 64, 288)])
def test_product_with_k_split(cuda_dev, fmt, split, M, N, K):
    """Single-CTA tiles with K shared by a cluster, stages divided evenly or not."""
    _, xq = make_rows(M, K, fmt, torch.bfloat16, 3, cuda_dev)
    _, wq = make_rows(N, K, fmt, torch.bfloat16, 4, cuda_dev)
    bias = torch.randn(N, device=cuda_dev)
    _lib.set_option("fp4_pair", 0)
    _lib.set_option("fp4_split", split)
    y = fp4_exec.fp4_gemm(xq, wq, bias, torch.float16)
    check_product(y, xq, wq, bias, fmt)
    assert torch.equal(fp4_exec.fp4_gemm(xq, wq, bias, torch.float16), y)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("M,N,K", [(2048, 640, 640), (5000, 100, 160), (20000, 60, 96)])
def test_product_more_single_tiles_than_sms(cuda_dev, fmt, M, N, K):
    g = torch.Generator().manual_seed(8)
    xq = fp4_exec.quant_rows_fp4(torch.randn(M, K, generator=g).to(torch.bfloat16).to(cuda_dev), fmt)
    wq = fp4_exec.quant_rows_fp4(torch.randn(N, K, generator=g).to(torch.bfloat16).to(cuda_dev), fmt)
    _lib.set_option("fp4_pair", 0)
    check_product(fp4_exec.fp4_gemm(xq, wq, None, torch.bfloat16), xq, wq, None, fmt)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("M,N,K,bias", [(256, 256, 64, False), (1, 8, 32, True), (300, 520, 288, True), (129, 640, 2592, False),
                                        (520, 264, 1280, True), (2300, 2312, 96, True), (3000, 2560, 1600, False), (4173, 640, 2560, True), (700, 333, 160, True), (257, 257, 64, False)])
def test_product_on_cta_pairs(cuda_dev, fmt, M, N, K, bias):
    """The CTA-pair kernel at sizes below and above one tile per pair, ragged in every direction."""
    g = torch.Generator().manual_seed(M + N)
    x = torch.randn(M, K, generator=g).to(torch.float16).to(cuda_dev)
    w = torch.randn(N, K, generator=g).to(torch.bfloat16).to(cuda_dev)
    xq, wq = fp4_exec.quant_rows_fp4(x, fmt), fp4_exec.quant_rows_fp4(w, fmt)
    b = torch.randn(N, generator=g).to(cuda_dev) if bias else None
    _lib.set_option("fp4_pair", 2)
    try:
        y = fp4_exec.fp4_gemm(xq, wq, b, torch.float16)
        again = fp4_exec.fp4_gemm(xq, wq, b, torch.float16)
    finally:
        _lib.set_option("fp4_pair", 1)
    check_product(y, xq, wq, b, fmt)
    assert torch.equal(y, again)


# ------------------------------------------------------------------------------------------------ product with a low-rank term
def low_rank_case(M, N, K, fmt, dtype, dev):
    """Packed operands, t = x A in ``dtype``, B and the fp32 factors that the product takes."""
    x, xq = make_rows(M, K, fmt, dtype, 1, dev)
    _, wq = make_rows(N, K, fmt, torch.bfloat16, 2, dev)
    g = torch.Generator().manual_seed(K + N)
    fi = torch.finfo(dtype)
    t = (x.double() @ (torch.randn(K, 32, generator=g).double() / K ** 0.5).to(dev)).clamp(-fi.max, fi.max).to(dtype)
    B = (torch.randn(32, N, generator=g) / 3).to(dtype).to(dev)
    return xq, wq, t, B, (fp4_exec.lowrank_rows(t, xq), fp4_exec.lowrank_weight(B, wq))


def check_low_rank(y, xq, wq, bias, fmt, t, B):
    """As check_product with 32 terms more.  The factors are exact in TF32 (16-bit values over powers of two), their products in
    fp32; each of the 32 additions is off by at most 2^-23 of the sum of magnitudes."""
    X, W = (ofp4.packed_values(q.codes.cpu(), q.scales.cpu(), None if q.row_scale is None else q.row_scale.cpu(), fmt) for q in (xq, wq))
    K = X.shape[1]
    T, U = t.cpu().double(), B.cpu().double()
    ref = X @ W.t() + T @ U
    S = X.abs() @ W.abs().t() + T.abs() @ U.abs()
    bound = (K / 16 + 36) * 2.0 ** -23 * S
    if bias is not None:
        ref = ref + bias.cpu().double()
        bound = bound + 2.0 ** -24 * (S + bias.cpu().double().abs())
    fi = torch.finfo(y.dtype)
    bound = bound + (ref.abs() + bound) * fi.eps / 2 + fi.smallest_normal * fi.eps / 2
    border = fi.max * (2 - fi.eps / 2) / (2 - fi.eps)
    got = y.cpu().double()
    inside = ref.abs() + bound < border
    assert bool(torch.isfinite(got[inside]).all()) and torch.equal(got[ref.abs() - bound >= border].abs(), torch.full_like(got[ref.abs() - bound >= border], float("inf")))
    worst = float((torch.where(inside, (got - ref).abs(), torch.zeros_like(ref)) / bound).max())
    assert worst <= 1, f"error {worst:.3g} times the bound"


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,N,K,options", [(1, 8, 32, {}), (5, 7, 96, {}), (128, 64, 256, {}), (77, 200, 640, {}), (129, 131, 288, {}),
                                           (1, 1280, 5120, {}), (33, 650, 2592, {"fp4_pair": 0, "fp4_split": 8}),
                                           (300, 200, 1280, {"fp4_pair": 0, "fp4_split": 2}), (2500, 587, 64, {"fp4_pair": 0}),
                                           (1300, 2056, 2080, {"fp4_pair": 0}), (256, 256, 64, {"fp4_pair": 2}), (1, 8, 32, {"fp4_pair": 2}),
                                           (300, 520, 288, {"fp4_pair": 2}), (2300, 2312, 96, {"fp4_pair": 2}),
                                           (3000, 2560, 1600, {"fp4_pair": 2}), (700, 333, 160, {"fp4_pair": 2}), (4173, 640, 2560, {})])
def test_product_with_a_low_rank_term(cuda_dev, fmt, dtype, M, N, K, options):
    xq, wq, t, B, factors = low_rank_case(M, N, K, fmt, dtype, cuda_dev)
    assert torch.equal(factors[0].double() * (1 if fmt == "mx" else xq.row_scale.double()[:, None]), t.double())
    assert torch.equal(factors[1].double() * (1 if fmt == "mx" else wq.row_scale.double()[:, None]), B.t().double())
    bias = torch.randn(N, device=cuda_dev) if N % 3 else None
    for k, v in options.items():
        _lib.set_option(k, v)
    try:
        y = fp4_exec.fp4_gemm(xq, wq, bias, dtype, factors)
        again = fp4_exec.fp4_gemm(xq, wq, bias, dtype, factors)
        nothing = fp4_exec.fp4_gemm(xq, wq, bias, dtype, (torch.zeros_like(factors[0]), factors[1]))
        plain = fp4_exec.fp4_gemm(xq, wq, bias, dtype)
    finally:
        _lib.set_option("fp4_pair", 1)
        _lib.set_option("fp4_split", 0)
    check_low_rank(y, xq, wq, bias, fmt, t, B)
    assert torch.equal(y, again) and torch.equal(nothing, plain)


@pytest.mark.parametrize("fmt", FMTS)
def test_low_rank_refusals_and_layouts(cuda_dev, fmt):
    xq, wq, t, B, (tl, lb) = low_rank_case(40, 72, 96, fmt, torch.bfloat16, cuda_dev)
    want = fp4_exec.fp4_gemm(xq, wq, None, torch.bfloat16, (tl, lb))
    wide = torch.zeros(40, 40, device=cuda_dev, dtype=torch.bfloat16)
    wide[:, 3:35] = t
    assert torch.equal(fp4_exec.lowrank_rows(wide[:, 3:35], xq), tl)             # rows that are not contiguous are copied
    assert fp4_exec.lowrank_rows(t[:0], fp4_exec.Fp4Rows(xq.codes[:0], xq.scales[:0], None if fmt == "mx" else xq.row_scale[:0])).shape == (0, 32)
    for bad in ((tl[:39], lb), (tl, lb[:, :31]), (tl.half(), lb), (tl.cpu(), lb), (tl, lb.t().contiguous().t()), (tl, None)):
        with pytest.raises(AssertionError):
            fp4_exec.fp4_gemm(xq, wq, None, torch.bfloat16, bad)
    for bad in (t[:, :16], t.float().cpu(), t[None]):
        with pytest.raises((AssertionError, TypeError)):
            fp4_exec.lowrank_rows(bad, xq)
    with pytest.raises(AssertionError):
        fp4_exec.lowrank_weight(B[:, :71], wq)
    assert torch.equal(torch.ops.pq_b200.fp4_gemm(xq.codes, xq.scales, xq.row_scale, wq.codes, wq.scales, wq.row_scale, None, 0, tl, lb), want)
    assert torch.equal(torch.ops.pq_b200.fp4_lowrank_rows(t, xq.row_scale), tl)


@pytest.mark.parametrize("fmt", FMTS)
def test_low_rank_general_path_agrees_with_the_one_step_calls(cuda_dev, fmt, monkeypatch):
    xq, wq, t, B, (tl, lb) = low_rank_case(90, 136, 288, fmt, torch.bfloat16, cuda_dev)
    bias = torch.randn(136, device=cuda_dev)
    bind = ops._BIND()
    status = ops.status_word(tl.device).data_ptr(), _lib.GEMM_WORKSPACE_BYTES
    assert bind.fp4_lowrank_rows(t, xq.row_scale) is not None
    assert bind.fp4_gemm(*xq, *wq, bias, True, *status, tl, lb) is not None
    for bad in ((tl, None), (tl[:89], lb), (tl, lb.double()), (tl[:, ::2], lb), (tl, lb.t().contiguous().t())):
        assert bind.fp4_gemm(*xq, *wq, bias, True, *status, *bad) is None
    for bad in ((t.float(), xq.row_scale), (t[:, :16], xq.row_scale), (t, torch.ones(89, device=cuda_dev)), (t.t().contiguous().t(), None)):
        assert bind.fp4_lowrank_rows(*bad) is None
    one = fp4_exec.fp4_gemm(xq, wq, bias, torch.float16, (tl, lb))

    class Refuses:
        def __getattr__(self, name):
            return lambda *a: None
    monkeypatch.setattr(ops, "_bind_handle", Refuses())
    assert torch.equal(fp4_exec.lowrank_rows(t, xq), tl) and torch.equal(fp4_exec.fp4_gemm(xq, wq, bias, torch.float16, (tl, lb)), one)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("dtype", DTYPES)
def test_linear_with_a_low_rank_branch(cuda_dev, fmt, dtype):
    """Rank 32 goes through the product's accumulator, other ranks after it; the laid-out factor follows the buffers."""
    torch.manual_seed(4)
    lin = nn.Linear(640, 328).to(dtype)
    x = torch.randn(75, 640, device=cuda_dev).to(dtype)
    A, B = (torch.randn(640, 32) / 25).to(dtype), (torch.randn(32, 328) / 5).to(dtype)
    m = fp4_exec.Fp4Linear(lin, device=cuda_dev, fmt=fmt, lowrank=(A, B))
    xq = fp4_exec.quant_rows_fp4(x, fmt)

    def want():
        t = m._down(x)
        return fp4_exec.fp4_gemm(xq, m.weight_rows, m.bias, dtype, (fp4_exec.lowrank_rows(t, xq), fp4_exec.lowrank_weight(m.lr_B, m.weight_rows)))
    first = m(x)
    assert torch.equal(first, want())
    check_low_rank(first, xq, m.weight_rows, m.bias, fmt, m._down(x), m.lr_B)
    m.lr_B.mul_(-2)                                               # written in place
    assert torch.equal(m(x), want()) and not torch.equal(m(x), first)
    m.lr_B = torch.ones_like(m.lr_B)                              # replaced
    assert torch.equal(m(x), want())
    if m.weight_row_scale is not None:
        m.weight_row_scale.mul_(2)
        assert torch.equal(m(x), want())
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    m.lr_B.mul_(0.5)                                              # laid out anew inside the capture
    with torch.cuda.graph(graph):
        y = m(x)
    graph.replay()
    assert torch.equal(y, want())
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        z = m(x)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(z, want())
    assert m(x[:0]).shape == (0, 328) and torch.equal(m(x[0]), m(x[:1])[0])
    other = fp4_exec.Fp4Linear(lin, device=cuda_dev, fmt=fmt, lowrank=(A[:, :16].contiguous(), B[:16].contiguous()))
    ref = fp4_exec.fp4_gemm(xq, other.weight_rows, other.bias, dtype)
    assert torch.equal(other(x), torch.addmm(ref, x @ other.lr_A, other.lr_B))


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("pair", [1, 2])
def test_product_leaves_its_neighbourhood_alone(cuda_dev, fmt, pair):
    """Rows behind the last one, columns behind the last one and the bytes around the output stay as they were."""
    M, N, K = 70, 90, 128
    _lib.set_option("fp4_pair", pair)
    _, xq = make_rows(M, K, fmt, torch.bfloat16, 1, cuda_dev)
    _, wq = make_rows(N, K, fmt, torch.bfloat16, 2, cuda_dev)
    want = fp4_exec.fp4_gemm(xq, wq, None, torch.bfloat16)
    lib = _lib.load()
    for ldo, off in ((96, 0), (96, 8), (91, 1)):
        buf = torch.full((80 * 96,), 7.0, dtype=torch.bfloat16, device=cuda_dev)
        p = lambda t: None if t is None else t.data_ptr()       # noqa: E731
        rc = lib.pq_fp4_gemm(p(xq.codes), K // 2, p(xq.scales), p(xq.row_scale), p(wq.codes), K // 2, p(wq.scales), p(wq.row_scale),
                             None, ops.FP4_FORMATS[fmt], buf.data_ptr() + 2 * off, 0, ldo, M, N, K, None, 0,
                             torch.cuda.current_stream().cuda_stream)
        assert rc == 0
        got = buf[off: off + M * ldo].view(M, ldo)
        assert torch.equal(got[:, :N], want)
        got[:, :N] = 7.0
        assert bool((buf == 7.0).all())
    _lib.set_option("fp4_pair", 1)


@pytest.mark.parametrize("M,N,K,options", [(130, 1, 96, {"fp4_pair": 0}), (70, 131, 96, {"fp4_pair": 0}), (2500, 587, 64, {"fp4_pair": 0}),
                                           (33, 67, 1280, {"fp4_pair": 0, "fp4_split": 4}), (1, 63, 1280, {"fp4_pair": 0, "fp4_split": 2}),
                                           (290, 577, 96, {"fp4_pair": 2}), (290, 263, 96, {"fp4_pair": 2})])
def test_product_rows_at_every_border(cuda_dev, M, N, K, options):
    """Rows of odd length, odd stride and odd start in every variant: exactly the outputs are written."""
    _, xq = make_rows(M, K, "mx", torch.bfloat16, 1, cuda_dev)
    _, wq = make_rows(N, K, "mx", torch.bfloat16, 2, cuda_dev)
    lib = _lib.load()
    for k, v in options.items():
        _lib.set_option(k, v)
    try:
        want = None
        for ldo, off in ((-(-N // 8) * 8, 8), (N, 0), (N + 1, 1), (N + 2, 2), (N + 3, 5)):
            buf = torch.full((M * ldo + 16,), 7.0, dtype=torch.float16, device=cuda_dev)
            rc = lib.pq_fp4_gemm(xq.codes.data_ptr(), K // 2, xq.scales.data_ptr(), None, wq.codes.data_ptr(), K // 2, wq.scales.data_ptr(),
                                 None, None, ops.FP4_FORMATS["mx"], buf.data_ptr() + 2 * off, 1, ldo, M, N, K, None, 0,
                                 torch.cuda.current_stream().cuda_stream)
            assert rc == 0
            got = buf[off: off + M * ldo].view(M, ldo)
            if want is None:
                want = got[:, :N].clone()
                check_product(want, xq, wq, None, "mx")
            assert torch.equal(got[:, :N], want)
            got[:, :N] = 7.0
            assert bool((buf == 7.0).all())
    finally:
        _lib.set_option("fp4_pair", 1)
        _lib.set_option("fp4_split", 0)


@pytest.mark.parametrize("fmt", FMTS)
def test_product_strided_codes_and_repeatability(cuda_dev, fmt):
    _, xq = make_rows(150, 1280, fmt, torch.bfloat16, 1, cuda_dev)
    _, wq = make_rows(200, 1280, fmt, torch.bfloat16, 2, cuda_dev)
    want = fp4_exec.fp4_gemm(xq, wq, None, torch.float16)
    wide = torch.full((150, 704), 0xAA, dtype=torch.uint8, device=cuda_dev)
    for off in (0, 16, 8):                                        # 8: copied first
        view = wide[:, off: off + 640]
        view.copy_(xq.codes)
        got = fp4_exec.fp4_gemm(fp4_exec.Fp4Rows(view, xq.scales, xq.row_scale), wq, None, torch.float16)
        assert torch.equal(got, want)
    for _ in range(5):
        assert torch.equal(fp4_exec.fp4_gemm(xq, wq, None, torch.float16), want)


@pytest.mark.parametrize("fmt", FMTS)
def test_general_path_agrees_with_the_one_step_calls(cuda_dev, fmt, monkeypatch):
    """Operands that the one-step calls refuse take the step-by-step path; both give the same bytes."""
    x, xq = make_rows(150, 640, fmt, torch.bfloat16, 1, cuda_dev)
    _, wq = make_rows(200, 640, fmt, torch.bfloat16, 2, cuda_dev)
    bias = torch.randn(200, device=cuda_dev)
    bind = ops._BIND()
    code = ops.FP4_FORMATS[fmt]
    assert bind.quant_rows_fp4(x, code) is not None
    for odd in (x.float(), x[:, ::2], x[:, 8:], x[:, :48], x[0], x.t()):
        assert bind.quant_rows_fp4(odd, code) is None
    assert bind.fp4_gemm(*xq, *wq, bias.double(), True, 0, 0) is None and bind.fp4_gemm(*xq, *wq, bias[1:], True, 0, 0) is None
    assert bind.fp4_gemm(xq.codes[:, ::2], *xq[1:], *wq, None, True, 0, 0) is None
    one = (fp4_exec.quant_rows_fp4(x, fmt), fp4_exec.dequant_rows_fp4(xq), fp4_exec.fp4_gemm(xq, wq, bias, torch.float16))
    class Refuses:
        def __getattr__(self, name):
            return lambda *a: None
    monkeypatch.setattr(ops, "_bind_handle", Refuses())
    step = (fp4_exec.quant_rows_fp4(x, fmt), fp4_exec.dequant_rows_fp4(xq), fp4_exec.fp4_gemm(xq, wq, bias, torch.float16))
    assert torch.equal(one[0].codes, step[0].codes) and torch.equal(one[1], step[1]) and torch.equal(one[2], step[2])


@pytest.mark.parametrize("fmt", FMTS)
def test_refusals(cuda_dev, fmt):
    x, xq = make_rows(8, 128, fmt, torch.bfloat16, 1, cuda_dev)
    _, wq = make_rows(16, 128, fmt, torch.bfloat16, 2, cuda_dev)
    _, other = make_rows(16, 128, "nv" if fmt == "mx" else "mx", torch.bfloat16, 2, cuda_dev)
    _, longer = make_rows(16, 160, fmt, torch.bfloat16, 2, cuda_dev)
    R = fp4_exec.Fp4Rows
    for bad in (lambda: fp4_exec.fp4_gemm(xq, other), lambda: fp4_exec.fp4_gemm(xq, longer),
                lambda: fp4_exec.fp4_gemm(R(xq.codes, wq.scales[:, :0], xq.row_scale), wq),
                lambda: fp4_exec.fp4_gemm(R(xq.codes.int(), xq.scales, xq.row_scale), wq),
                lambda: fp4_exec.fp4_gemm(xq, wq, torch.zeros(15, device=cuda_dev)),
                lambda: fp4_exec.fp4_gemm(xq, wq, torch.zeros(16, device=cuda_dev, dtype=torch.bfloat16)),
                lambda: fp4_exec.fp4_gemm(xq, wq, torch.zeros(16)),
                lambda: fp4_exec.quant_rows_fp4(x[:, :48], fmt)):
        with pytest.raises(AssertionError):
            bad()
    with pytest.raises(TypeError):
        fp4_exec.quant_rows_fp4(x.float(), fmt)
    with pytest.raises(TypeError):
        fp4_exec.fp4_gemm(xq, wq, None, torch.float32)
    with pytest.raises(ValueError):
        fp4_exec.quant_rows_fp4(x, "int4")


# ------------------------------------------------------------------------------------------------ the Linear
@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("dtype", DTYPES)
def test_linear_runs_its_operators(cuda_dev, fmt, dtype):
    torch.manual_seed(2)
    lin = nn.Linear(640, 328).to(dtype)
    A, B = (torch.randn(640, 32) / 25).to(dtype), (torch.randn(32, 328) / 5).to(dtype)
    m = fp4_exec.Fp4Linear(lin, device=cuda_dev, fmt=fmt)
    x = torch.randn(2, 75, 640, device=cuda_dev).to(dtype)
    y = m(x)
    xq = fp4_exec.quant_rows_fp4(x.reshape(-1, 640), fmt)
    assert y.shape == (2, 75, 328) and torch.equal(y.reshape(-1, 328), fp4_exec.fp4_gemm(xq, m.weight_rows, m.bias, dtype))
    check_product(y.reshape(-1, 328), xq, m.weight_rows, m.bias, fmt)
    low = fp4_exec.Fp4Linear(lin, device=cuda_dev, fmt=fmt, lowrank=(A, B))
    yl = low(x)
    ref = y.double() + ((x.double() @ A.to(cuda_dev).double()).to(dtype).double() @ B.to(cuda_dev).double())
    # y and the sum are rounded once each, x @ A once (its half step carried through B, 32 terms of |t| |B| <= about 4 * 1)
    eps = torch.finfo(dtype).eps
    assert float((yl.double() - ref).abs().max()) <= eps * (float(ref.abs().max()) + float(y.abs().max())) + eps * 32
    assert m(x[:, :0]).shape == (2, 0, 328)
    assert torch.equal(m(x[0, 0]), y[0, 0])


def test_streams_graphs_and_compile_wrappers(cuda_dev):
    torch.manual_seed(3)
    lin = nn.Linear(1280, 640).to(torch.bfloat16)
    m = fp4_exec.Fp4Linear(lin, device=cuda_dev, fmt="nv")
    x = torch.randn(300, 1280, device=cuda_dev).to(torch.bfloat16)
    want = m(x)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = m(x)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    with torch.cuda.stream(side):
        m(x)
    torch.cuda.synchronize()
    g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    xs = x.clone()
    with torch.cuda.graph(g1):
        y1 = m(xs)
    with torch.cuda.graph(g2):
        y2 = m(xs * 2)
    xs.copy_(x)
    g1.replay(); g2.replay()
    torch.cuda.synchronize()
    assert torch.equal(y1, want) and torch.equal(y2, m(x * 2))
    ops_ns = torch.ops.pq_b200
    c, s, r = ops_ns.quant_rows_fp4(x, "nv")
    assert torch.equal(ops_ns.fp4_gemm(c, s, r, *m.weight_rows, m.bias, 0), want)
    assert torch.equal(ops_ns.dequant_rows_fp4(c, s, r, 0), fp4_exec.dequant_rows_fp4(fp4_exec.quant_rows_fp4(x, "nv")))
    c, s, r = ops_ns.quant_rows_fp4(x, "mx")
    assert r.numel() == 0


@pytest.mark.parametrize("fmt", FMTS)
def test_rows_that_overlap(cuda_dev, fmt):
    """One row seen many times (a broadcast input) and windows that share elements are copied first, codes likewise."""
    x = awkward_rows(40, 320, torch.bfloat16, 6).to(cuda_dev)
    for view in (x[3:4].expand(70, 320), x.as_strided((20, 320), (64, 1)), x[:, :32][5:6].expand(3, 32)):
        check_rows(fp4_exec.quant_rows_fp4(view, fmt), view, fmt)
    q = fp4_exec.quant_rows_fp4(x[3:4].expand(70, 320), fmt)
    wq = fp4_exec.quant_rows_fp4(x, fmt)
    same = fp4_exec.Fp4Rows(q.codes[:1].expand(70, 160), q.scales, q.row_scale)
    assert torch.equal(fp4_exec.fp4_gemm(same, wq, None, torch.bfloat16).view(torch.int16),
                       fp4_exec.fp4_gemm(q, wq, None, torch.bfloat16).view(torch.int16))
    assert torch.equal(fp4_exec.dequant_rows_fp4(same).view(torch.int16), fp4_exec.dequant_rows_fp4(q).view(torch.int16))


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("M,N,K", [(1, 640, 640), (77, 1280, 640), (1000, 640, 2560), (4096, 1280, 640)])
def test_kernels_in_a_row_wait_for_one_another(cuda_dev, fmt, M, N, K):
    """Quantisation, product, read-back, group norm and product again, eager and replayed, on memory that every call takes over from
    the one before: the results of calls that are synchronised one by one."""
    from pyraquant_b200 import norm_exec
    g = torch.Generator().manual_seed(M + N)
    xs = [torch.randn(M, K, generator=g).to(torch.bfloat16).to(cuda_dev) for _ in range(3)]
    wq = fp4_exec.quant_rows_fp4(torch.randn(N, K, generator=g).to(torch.bfloat16).to(cuda_dev), fmt)
    b = torch.randn(N, generator=g).to(cuda_dev)
    gamma, beta = torch.randn(K, generator=g).to(cuda_dev).bfloat16(), torch.randn(K, generator=g).to(cuda_dev).bfloat16()

    def run(x, between):
        q = fp4_exec.quant_rows_fp4(x, fmt)
        between()
        y = fp4_exec.fp4_gemm(q, wq, b, torch.bfloat16)
        between()
        z = fp4_exec.dequant_rows_fp4(q, torch.bfloat16)
        between()
        n = norm_exec.group_norm_quant_fp4(z[None], 32, gamma, beta, 1e-5, "silu", fmt)
        between()
        return y, z, fp4_exec.fp4_gemm(n, wq, b, torch.bfloat16)

    want = [run(x, torch.cuda.synchronize) for x in xs]
    for _ in range(10):
        for x, w in zip(xs, want):
            got = run(x, lambda: None)
            assert all(torch.equal(a, e) for a, e in zip(got, w))
            del got
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = [run(x, lambda: None) for x in xs]
    for _ in range(5):
        graph.replay()
    torch.cuda.synchronize()
    for a, w in zip(got, want):
        assert all(torch.equal(u, e) for u, e in zip(a, w))


def test_several_threads_and_streams(cuda_dev):
    """Group norm, quantisation and products with a low-rank term from three threads at once, each on a stream of its own."""
    import threading

    from pyraquant_b200 import norm_exec
    torch.manual_seed(7)
    shapes = [(2, 1024, 640, 640, "mx"), (1, 4096, 320, 1280, "nv"), (3, 77, 1280, 200, "nv")]

    def make(B, T, C, N, fmt):
        x = torch.randn(B, T, C, device=cuda_dev).bfloat16()
        w = torch.randn(C, device=cuda_dev).bfloat16()
        W = fp4_exec.quant_rows_fp4(torch.randn(N, C, device=cuda_dev).bfloat16(), fmt)
        t = torch.randn(B * T, 32, device=cuda_dev).bfloat16()
        lb = fp4_exec.lowrank_weight(torch.randn(32, N, device=cuda_dev).bfloat16(), W)

        def run():
            z = norm_exec.group_norm_rows(x, 32, w, w, 1e-5, "silu")
            q = norm_exec.group_norm_quant_fp4(x, 32, w, w, 1e-5, "silu", fmt)
            y = fp4_exec.fp4_gemm(q, W, None, torch.bfloat16, (fp4_exec.lowrank_rows(t, q), lb))
            q2 = fp4_exec.quant_rows_fp4(z.reshape(-1, C), fmt)
            return y, fp4_exec.fp4_gemm(q2, W, None, torch.bfloat16), fp4_exec.dequant_rows_fp4(q2)
        return run
    runs = [make(*s) for s in shapes]
    want = [r() for r in runs]
    torch.cuda.synchronize()
    wrong = [None] * 3

    def worker(i):
        s = torch.cuda.Stream()
        n = 0
        with torch.cuda.stream(s):
            for _ in range(40):
                n += sum(not torch.equal(a, b) for a, b in zip(runs[i](), want[i]))
        wrong[i] = n
    threads = [threading.Thread(target=worker, args=(i,)) for i in range(3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert wrong == [0, 0, 0]


def test_linear_in_inference_mode(cuda_dev):
    """Weights made in inference mode and calls inside it give the values of ordinary ones."""
    torch.manual_seed(8)
    lin = nn.Linear(320, 96).to(torch.bfloat16)
    low = (torch.randn(320, 32) / 18).bfloat16(), (torch.randn(32, 96) / 5).bfloat16()
    x = torch.randn(9, 320, device=cuda_dev).bfloat16()
    want = fp4_exec.Fp4Linear(lin, device=cuda_dev, lowrank=low)(x)
    with torch.inference_mode():
        m = fp4_exec.Fp4Linear(lin, device=cuda_dev, lowrank=low)
        assert torch.equal(m(x), want)
        m.lr_B.mul_(2)                                            # nothing counts this change
        doubled = m(x)
    assert not torch.equal(doubled, want) and torch.equal(m(x), doubled)


@pytest.mark.parametrize("fmt,K", [("nv", 2 ** 28 + 64), ("mx", 2 ** 29 + 128)])
def test_rows_whose_scales_pass_two_gigabytes(cuda_dev, fmt, K):
    """Offsets into the scale tiles of one row need more than 31 bits."""
    x = torch.zeros(1, K, dtype=torch.bfloat16, device=cuda_dev)
    ends = awkward_rows(1, 256, torch.bfloat16, 12).to(cuda_dev)
    x[:, :128], x[:, -128:] = ends[:, :128], ends[:, 128:]
    q = fp4_exec.quant_rows_fp4(x, fmt)
    assert q.scales.numel() > 2 ** 31
    v = fp4_exec.dequant_rows_fp4(q)
    small = fp4_exec.dequant_rows_fp4(fp4_exec.quant_rows_fp4(ends, fmt))
    assert torch.equal(v[:, :128], small[:, :128]) and torch.equal(v[:, -128:], small[:, 128:])
    assert not v[:, 128:-128].any()


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("dtype", DTYPES)
def test_read_back_of_every_magnitude(cuda_dev, fmt, dtype):
    """Finite rows come back finite, the type's largest among them, and as the values of their codes."""
    top = 0x7F80 if dtype == torch.bfloat16 else 0x7C00
    v = torch.arange(1, top, dtype=torch.int32).to(torch.int16).view(dtype)
    x = torch.stack([v * f for f in (1.0, 0.75, -0.4, -1.0)], dim=1).repeat(1, 8)
    q = fp4_exec.quant_rows_fp4(x.to(cuda_dev), fmt)
    want = ofp4.packed_values(q.codes.cpu(), q.scales.cpu(), None if q.row_scale is None else q.row_scale.cpu(), fmt)
    for t in DTYPES:
        got, most = fp4_exec.dequant_rows_fp4(q, t).cpu(), torch.finfo(t).max
        assert bool(torch.isfinite(got).all()) and torch.equal(got, want.clamp(-most, most).to(t))
    assert dtype == torch.float16 or fmt == "mx" or bool((want.abs() > torch.finfo(dtype).max).any())


@pytest.mark.parametrize("op", ["quant", "dequant", "product", "factors", "norm", "norm_int8", "norm_fp4"])
def test_calls_let_other_threads_run(cuda_dev, op):
    """A launch waits while the queue is full.  Other Python threads run meanwhile."""
    import threading
    import time

    from pyraquant_b200 import norm_exec
    x = torch.randn(4, 64, device=cuda_dev).bfloat16()
    q, t, B = fp4_exec.quant_rows_fp4(x, "nv"), torch.randn(4, 32, device=cuda_dev).bfloat16(), torch.randn(32, 4, device=cuda_dev).bfloat16()
    call = {"quant": lambda: fp4_exec.quant_rows_fp4(x, "nv"), "dequant": lambda: fp4_exec.dequant_rows_fp4(q),
            "product": lambda: fp4_exec.fp4_gemm(q, q), "factors": lambda: fp4_exec.lowrank_factors(t, q, B, q),
            "norm": lambda: norm_exec.group_norm_rows(x[None], 4), "norm_int8": lambda: norm_exec.group_norm_quant_rows(x[None], 4),
            "norm_fp4": lambda: norm_exec.group_norm_quant_fp4(x[None], 4)}[op]
    call()
    torch.cuda.synchronize()
    longest, stop = [0.0], threading.Event()

    def ticker():
        last = time.perf_counter()
        while not stop.is_set():
            time.sleep(0.002)
            now = time.perf_counter()
            longest[0], last = max(longest[0], now - last), now
    other = threading.Thread(target=ticker)
    other.start()
    waited = 0.0
    try:
        torch.cuda._sleep(1_200_000_000)                          # some 0.6 s
        for _ in range(4000):
            t0 = time.perf_counter()
            call()
            waited = max(waited, time.perf_counter() - t0)
            if waited > 0.1:
                break
    finally:
        stop.set()
        other.join()
        torch.cuda.synchronize()
    assert waited > 0.1, "no call had to wait"
    assert longest[0] < waited / 2, (longest[0], waited)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("dtype", DTYPES)
def test_linear_2d(cuda_dev, fmt, dtype):
    x = awkward_rows(77, 640, dtype, 3).to(cuda_dev)
    w = fp4_exec.quant_rows_fp4(awkward_rows(200, 640, torch.bfloat16, 4).to(cuda_dev), fmt)
    b = torch.randn(200, device=cuda_dev)
    y = fp4_exec.fp4_linear_2d(x, w, b)
    assert y.dtype == dtype and torch.equal(y, fp4_exec.fp4_gemm(fp4_exec.quant_rows_fp4(x, fmt), w, b, dtype))
    check_product(y, fp4_exec.quant_rows_fp4(x, fmt), w, b, fmt)
    m = fp4_exec.Fp4Linear(nn.Linear(640, 200).to(dtype), device=cuda_dev, fmt=fmt)
    assert torch.equal(m(x), fp4_exec.fp4_linear_2d(x, m.weight_rows, m.bias))


def test_graph_of_two_branches(cuda_dev):
    """Capture over two streams that part and meet again: the chained launches behind the meeting wait for both."""
    g = torch.Generator().manual_seed(4)
    x, u = (torch.randn(300, 640, generator=g).bfloat16().to(cuda_dev) for _ in range(2))
    w = fp4_exec.quant_rows_fp4(torch.randn(640, 640, generator=g).bfloat16().to(cuda_dev), "nv")
    side = torch.cuda.Stream()

    def run():
        main = torch.cuda.current_stream()
        side.wait_stream(main)
        a = fp4_exec.quant_rows_fp4(x, "nv")
        with torch.cuda.stream(side):
            b = fp4_exec.quant_rows_fp4(u * 2, "nv")
            y1 = fp4_exec.fp4_gemm(b, w, None, torch.bfloat16)
        y0 = fp4_exec.fp4_gemm(a, w, None, torch.bfloat16)
        main.wait_stream(side)
        q = fp4_exec.quant_rows_fp4(y1, "nv")
        z = fp4_exec.fp4_gemm(q, w, None, torch.bfloat16)
        keep.append((a, b, q))
        return y0, y1, z
    keep = []
    want = run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run()
    for k in range(3):
        x.mul_(-1); u.mul_(-1)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, run() if k < 2 else [-t for t in want]):
            assert torch.equal(a, b)
