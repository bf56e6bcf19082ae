"""Group norm over channels-last rows against the formula in 64 bits, and its quantising forms against their parts.

Bound.  A thread sums at most L rows of x - pivot one after the other (L <= 64 for the sizes here) and at most 64 merges
follow: the mean is off by at most (L + 64) 2^-24 mean|x - pivot|, with |x - pivot| taken as at most 8 deviations, plus
one rounding of its own size, 2^-24 |mean| a few times over; the variance likewise, relative to itself.  So x-hat is off by
A (1 + |x-hat|) + 4 2^-24 |mean| / std with A = 128 * 8 * 2^-24 (a unit of the last term goes to the product of mean and
slope, which is rounded into the added constant).  gamma multiplies that, SiLU's slope is at most 1.1 and its own
evaluation, z / (1 + 2^t) with t = -z log2(e) and one reciprocal for two denominators, loses (in units of 2^-24): 1 + |z| (t rounds)
and 4 (exponential) in 2^t, 1 in the denominator that does not cancel, 1 in the product of the two, 2 in the reciprocal, 1 + 1 in
the products with it: (11 + |z|) 2^-24 of the value.  The
rounding to 16 bits is eps / 2 of the value or half the smallest subnormal.
"""
import ctypes

import pytest
import torch
import torch.nn as nn

from pyraquant_b200 import _lib, fp4_exec, int8_exec, norm_exec, ops

DTYPES = [torch.bfloat16, torch.float16]
A = 128 * 8 * 2.0 ** -24


def formula(x, groups, w, b, eps, act):
    """(z, bound before the rounding to 16 bits) in 64 bits; x [B, T, C]."""
    B, T, C = x.shape
    v = x.double().reshape(B, T, groups, C // groups)
    mean = v.mean(dim=(1, 3), keepdim=True)
    var = ((v - mean) ** 2).mean(dim=(1, 3), keepdim=True)
    rstd = 1 / torch.sqrt(var + eps)
    xh = (v - mean) * rstd
    # with eps > 0 the error of x-hat scales with rstd, not 1 / std
    err = (A * (torch.sqrt(var) * rstd + xh.abs()) + 4 * 2.0 ** -24 * mean.abs() * rstd).expand_as(v)
    w = torch.ones(C, dtype=torch.float64) if w is None else w.double()
    b = torch.zeros(C, dtype=torch.float64) if b is None else b.double()
    z = xh.reshape(B, T, C) * w + b
    err = err.reshape(B, T, C) * w.abs() + 2.0 ** -23 * (z.abs() + b.abs())
    if act == "silu":
        z, err = z / (1 + torch.exp(-z)), 1.1 * err + (11 + z.abs()) * 2.0 ** -24 * (z / (1 + torch.exp(-z))).abs()
    return z, err


def check(got, x, groups, w, b, eps, act):
    C = x.shape[-1]
    z, err = formula(x.cpu().reshape(x.shape[0], -1, C), groups, None if w is None else w.cpu(), None if b is None else b.cpu(), eps, act)
    fi = torch.finfo(got.dtype)
    bound = err + (z.abs() + err) * fi.eps / 2 + fi.smallest_normal * fi.eps / 2
    off = (got.cpu().double().reshape(z.shape) - z).abs()
    assert bool(torch.isfinite(got).all())
    worst = float((off / bound).max())
    assert worst <= 1, f"{worst:.3g} times the bound"


def rows(B, T, C, dtype, seed, mean=0.5):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(B, T, C, generator=g) * (0.3 + torch.rand(C, generator=g)) + mean * torch.randn(C, generator=g)
    return x.to(dtype), (1 + 0.3 * torch.randn(C, generator=g)).to(dtype), (0.3 * torch.randn(C, generator=g)).to(dtype)


SHAPES = [(1, 1, 8, 1), (2, 1, 32, 32), (1, 7, 64, 4), (3, 50, 320, 32), (1, 1000, 1280, 32), (2, 333, 640, 32), (1, 4097, 256, 32),
          (1, 100, 8192, 8), (1, 40, 4104, 3), (300, 3, 32, 4), (149, 2, 64, 8), (4, 2048, 128, 32), (1, 5, 1920, 32), (5, 601, 960, 32)]


@pytest.mark.gpu
@pytest.mark.parametrize("B,T,C,groups", SHAPES)
@pytest.mark.parametrize("dtype", DTYPES)
def test_group_norm(cuda_dev, dtype, B, T, C, groups):
    x, w, b = (t.to(cuda_dev) for t in rows(B, T, C, dtype, B + T + C))
    for act in (None, "silu"):
        check(norm_exec.group_norm_rows(x, groups, w, b, 1e-6, act), x, groups, w, b, 1e-6, act)
    check(norm_exec.group_norm_rows(x, groups), x, groups, None, None, 1e-6, None)
    check(norm_exec.group_norm_rows(x, groups, w.float(), b, 1e-5, "silu"), x, groups, w.float(), b, 1e-5, "silu")
    check(norm_exec.group_norm_rows(x, groups, None, b.float()), x, groups, None, b.float(), 1e-6, None)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_large_mean_and_outliers(cuda_dev, dtype):
    """A mean far above the deviation, rows that begin with an outlier (the pivot of the sums), constant groups."""
    g = torch.Generator().manual_seed(8)
    x = (100 + torch.randn(2, 600, 64, generator=g)).to(dtype)
    x[:, ::97] = 90
    x[1, :, :16] = 3.0                                            # variance 0
    check(norm_exec.group_norm_rows(x.to(cuda_dev), 8), x, 8, None, None, 1e-6, None)


@pytest.mark.gpu
def test_layouts(cuda_dev):
    x, w, b = (t.to(cuda_dev) for t in rows(3, 64, 320, torch.bfloat16, 4))
    want = norm_exec.group_norm_rows(x, 32, w, b)
    img = x.reshape(3, 8, 8, 320)
    assert torch.equal(norm_exec.group_norm_rows(img, 32, w, b), want.reshape(img.shape))
    nchw = img.permute(0, 3, 1, 2)                                # a channels_last image
    assert torch.equal(norm_exec.group_norm_rows(nchw.permute(0, 2, 3, 1), 32, w, b), want.reshape(img.shape))
    wide = torch.randn(3, 70, 400, device=cuda_dev).to(torch.bfloat16)
    for off in (0, 8, 3):                                         # 3: copied first
        view = wide[:, 2:66, off: off + 320]
        view.copy_(x)
        keep = wide.clone()
        assert torch.equal(norm_exec.group_norm_rows(view, 32, w, b), want)
        assert torch.equal(wide, keep)
    assert torch.equal(norm_exec.group_norm_rows(x[:1].expand(4, 64, 320), 32, w, b), want[:1].expand(4, 64, 320))
    assert torch.equal(norm_exec.group_norm_rows(x.transpose(1, 2).contiguous().transpose(1, 2), 32, w, b), want)
    assert norm_exec.group_norm_rows(x[:0], 32, w, b).shape == (0, 64, 320)
    assert norm_exec.group_norm_rows(x[:, :0], 32, w, b).shape == (3, 0, 320)
    odd = torch.randn(700, device=cuda_dev).to(torch.bfloat16)
    odd[3:323], odd[323:643] = w, b                                # affine vectors off 16-byte borders, and strided ones
    assert torch.equal(norm_exec.group_norm_rows(x, 32, odd[3:323], odd[323:643]), want)
    assert torch.equal(norm_exec.group_norm_rows(x, 32, torch.stack([w, b], 1)[:, 0], torch.stack([w, b], 1)[:, 1]), want)
    flat = torch.randn(5, 64, device=cuda_dev).to(torch.float16)   # [B, C]: one row per sample
    assert torch.equal(norm_exec.group_norm_rows(flat, 4), norm_exec.group_norm_rows(flat[:, None], 4)[:, 0])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,T,C,groups", [(1, 30000, 640, 32), (3, 4000, 1536, 32), (2, 1500, 8192, 16)])
def test_more_rows_than_the_chip_holds(cuda_dev, dtype, B, T, C, groups):
    """Rows beyond shared memory are read twice; the quantising forms fall back to two launches."""
    x, w, b = (t.to(cuda_dev) for t in rows(B, T, C, dtype, 11))
    z = norm_exec.group_norm_rows(x, groups, w, b, 1e-6, "silu")
    check(z, x, groups, w, b, 1e-6, "silu")
    assert torch.equal(norm_exec.group_norm_rows(x, groups, w, b, 1e-6, "silu"), z)
    q, s, zz = norm_exec.group_norm_quant_rows(x, groups, w, b, 1e-6, "silu", want_normed=True)
    q0, s0 = int8_exec.quant_rows(z.reshape(-1, C))
    assert torch.equal(zz, z) and torch.equal(q, q0) and torch.equal(s, s0)
    wide = torch.zeros(B, T, C + 64, device=cuda_dev, dtype=dtype)
    wide[..., 32: 32 + C] = x
    assert torch.equal(norm_exec.group_norm_rows(wide[..., 32: 32 + C], groups, w, b, 1e-6, "silu"), z)


@pytest.mark.gpu
def test_nan_stays_in_its_group(cuda_dev):
    x, w, b = (t.to(cuda_dev) for t in rows(2, 300, 64, torch.float16, 5))
    want = norm_exec.group_norm_rows(x, 8, w, b)
    x[1, 17, 20] = float("nan")
    got = norm_exec.group_norm_rows(x, 8, w, b)
    assert torch.isnan(got[1, :, 16:24]).all()
    got[1, :, 16:24] = want[1, :, 16:24]
    assert torch.equal(got, want)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,T,C", [(1, 1, 32), (2, 77, 320), (3, 250, 640), (1, 1024, 1280), (2, 40, 2560), (1, 9, 8192), (150, 2, 64), (400, 3, 96),
                                   (2, 3000, 224)])
def test_quantising_forms(cuda_dev, dtype, B, T, C):
    """The forms that quantise in the same call give the codes of the separate steps, bit for bit."""
    groups = 32 if C >= 320 else 4
    assert ops.group_norm_quant_rows_fused(torch.zeros(B, T, C, device=cuda_dev, dtype=dtype), groups, None, None, 1e-6, None, False) is not None
    x, w, b = (t.to(cuda_dev) for t in rows(B, T, C, dtype, 3 * C + T))
    for act in (None, "silu"):
        z = norm_exec.group_norm_rows(x, groups, w, b, 1e-6, act)
        q0, s0 = int8_exec.quant_rows(z.reshape(-1, C))
        for want_normed in (False, True):
            q, s, zz = norm_exec.group_norm_quant_rows(x, groups, w, b, 1e-6, act, want_normed=want_normed)
            assert torch.equal(q, q0) and torch.equal(s, s0)
            assert zz is None if not want_normed else torch.equal(zz, z)
        for fmt in ("mx", "nv"):
            f0, f = fp4_exec.quant_rows_fp4(z.reshape(-1, C), fmt), norm_exec.group_norm_quant_fp4(x, groups, w, b, 1e-6, act, fmt)
            assert f.fmt == fmt and torch.equal(f.codes, f0.codes)
            assert torch.equal(fp4_exec.dequant_rows_fp4(f), fp4_exec.dequant_rows_fp4(f0))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_in_front_of_a_linear(cuda_dev, dtype):
    torch.manual_seed(4)
    lin = nn.Linear(640, 640).to(dtype)
    low = ((torch.randn(640, 32) / 25).to(dtype), (torch.randn(32, 640) / 6).to(dtype))
    x, w, b = (t.to(cuda_dev) for t in rows(2, 90, 640, dtype, 6))
    x = x.reshape(2, 9, 10, 640)
    z = norm_exec.group_norm_rows(x, 32, w, b)
    for layer in (int8_exec.Int8Linear(lin, device=cuda_dev), int8_exec.Int8Linear(lin, device=cuda_dev, lowrank=low)):
        want = layer(z)
        y, zz = layer.forward_group_norm(x, 32, w, b, return_normed=True)
        assert y.shape == (2, 9, 10, 640) and torch.equal(zz, z)
        # the low-rank branch may be summed in another order by the one-launch prologue: a rounding of t, then of y
        tol = 0 if layer.lr_A is None else 4 * torch.finfo(dtype).eps * float(want.abs().max())
        assert float((y.float() - want.float()).abs().max()) <= tol
        assert torch.equal(layer.forward_group_norm(x, 32, w, b), y)
    for fmt in ("mx", "nv"):
        for layer in (fp4_exec.Fp4Linear(lin, device=cuda_dev, fmt=fmt), fp4_exec.Fp4Linear(lin, device=cuda_dev, fmt=fmt, lowrank=low)):
            assert torch.equal(layer.forward_group_norm(x, 32, w, b), layer(z))
    ops.check_device_status(cuda_dev)


@pytest.mark.gpu
def test_general_path_agrees_with_the_one_step_calls(cuda_dev, monkeypatch):
    x, w, b = (t.to(cuda_dev) for t in rows(2, 300, 320, torch.float16, 9))
    calls = (lambda: norm_exec.group_norm_rows(x, 32, w, b, 1e-6, "silu"),
             lambda: norm_exec.group_norm_quant_rows(x, 32, w, b, want_normed=True),
             lambda: norm_exec.group_norm_quant_fp4(x, 32, w, b, fmt="nv"), lambda: norm_exec.group_norm_quant_fp4(x, 32, None, b, fmt="mx"))
    one = [c() for c in calls]

    class Refuses:
        def __getattr__(self, name):
            return lambda *a: None
    monkeypatch.setattr(ops, "_bind_handle", Refuses())
    for a, c in zip(one, calls):
        s = c()
        if isinstance(a, torch.Tensor):
            assert torch.equal(a, s)
        elif isinstance(a, fp4_exec.Fp4Rows):
            assert torch.equal(fp4_exec.dequant_rows_fp4(fp4_exec.Fp4Rows(*(t if t is None else t.clone() for t in a))).float(), _values(s))
        else:
            assert all(torch.equal(p, q) for p, q in zip(a, s))


def _values(q):
    from oracle import fp4 as ofp4
    v = ofp4.packed_values(q.codes.cpu(), q.scales.cpu(), None if q.row_scale is None else q.row_scale.cpu(), q.fmt)
    return v.to(torch.bfloat16).float().to(q.codes.device)


@pytest.mark.gpu
def test_streams_graphs_and_repeats(cuda_dev):
    x, w, b = (t.to(cuda_dev) for t in rows(2, 5000, 320, torch.bfloat16, 7))
    want = norm_exec.group_norm_rows(x, 32, w, b, 1e-6, "silu")
    for _ in range(5):
        assert torch.equal(norm_exec.group_norm_rows(x, 32, w, b, 1e-6, "silu"), want)
    assert torch.equal(torch.ops.pq_b200.group_norm_rows(x, 32, w, b, 1e-6, True), want)
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    outs = []
    for i in range(12):
        with torch.cuda.stream(streams[i % 3]):
            outs.append(norm_exec.group_norm_rows(x, 32, w, b, 1e-6, "silu"))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)
    xs = x.clone()
    graphs, ys = [], []
    for k in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            ys.append(norm_exec.group_norm_quant_fp4(xs * (k + 1), 32, w, b, 1e-6, "silu", "nv"))
        graphs.append(g)
    for _ in range(3):
        for g in graphs:
            g.replay()
    torch.cuda.synchronize()
    for k in range(2):
        f0 = norm_exec.group_norm_quant_fp4(x * (k + 1), 32, w, b, 1e-6, "silu", "nv")
        assert torch.equal(ys[k].codes, f0.codes) and torch.equal(ys[k].row_scale, f0.row_scale)
    with torch.cuda.stream(streams[0]):
        graphs[0].replay()
    with torch.cuda.stream(streams[1]):
        graphs[1].replay()
    torch.cuda.synchronize()
    assert torch.equal(ys[1].codes, f0.codes)
    ops.check_device_status(cuda_dev)


@pytest.mark.gpu
def test_refusals_gpu(cuda_dev):
    x = torch.randn(2, 5, 64, device=cuda_dev).to(torch.bfloat16)
    for bad in (lambda: norm_exec.group_norm_rows(x, 7), lambda: norm_exec.group_norm_rows(x[..., :60], 4),
                lambda: norm_exec.group_norm_rows(x, 8, torch.ones(63, device=cuda_dev)), lambda: norm_exec.group_norm_rows(x, 8, torch.ones(64)),
                lambda: norm_exec.group_norm_rows(x, 8, torch.ones(64, device=cuda_dev, dtype=torch.float64)),
                lambda: norm_exec.group_norm_rows(torch.zeros(1, 1, 8200, device=cuda_dev, dtype=torch.float16), 1),
                lambda: norm_exec.group_norm_rows(x[0, 0], 8), lambda: norm_exec.group_norm_quant_fp4(x[..., :48].contiguous(), 4)):
        with pytest.raises(AssertionError):
            bad()
    with pytest.raises(TypeError):
        norm_exec.group_norm_rows(x.float(), 8)
    with pytest.raises(ValueError):
        norm_exec.group_norm_rows(x, 8, act="gelu")
    w = nn.Parameter(torch.ones(64, device=cuda_dev, dtype=torch.bfloat16))
    with pytest.raises(RuntimeError):
        norm_exec.group_norm_rows(x, 8, w)
    with torch.no_grad():
        norm_exec.group_norm_rows(x, 8, w)
    with torch.inference_mode():
        norm_exec.group_norm_rows(x, 8, w)


@pytest.mark.gpu
def test_refusals_of_the_traced_form(cuda_dev, monkeypatch):
    """Where a compiler traces the call, an unknown activation is refused too, and the known ones give the eager values."""
    x = torch.randn(2, 5, 64, device=cuda_dev).to(torch.bfloat16)
    want = {act: norm_exec.group_norm_rows(x, 8, act=act) for act in (None, "silu")}
    monkeypatch.setattr(norm_exec, "_eager", lambda: False)
    for act, z in want.items():
        assert torch.equal(norm_exec.group_norm_rows(x, 8, act=act), z)
    for f in (norm_exec.group_norm_rows, norm_exec.group_norm_quant_rows, norm_exec.group_norm_quant_fp4):
        with pytest.raises(ValueError):
            f(x, 8, act="gelu")


def test_refusals_on_the_host():
    with pytest.raises(AssertionError):
        norm_exec.group_norm_rows(torch.randn(2, 4, 64, dtype=torch.bfloat16), 8)


def test_argument_checks():
    lib = _lib.load()
    buf = ctypes.create_string_buffer(4096)
    p = (ctypes.addressof(buf) + 63) & ~63
    big = 1 << 30

    def gn(x=p, dtype=0, B=1, T=4, C=64, row=64, batch=256, groups=8, w=None, b=None, f32=0, eps=1e-6, act=0, out=p, orow=64,
           obatch=256, ws=p, wsb=big):
        return lib.pq_group_norm(x, dtype, B, T, C, row, batch, groups, w, b, f32, eps, act, out, orow, obatch, ws, wsb, None, None)
    assert gn(B=0, x=None) == 0 and gn(T=0, x=None) == 0
    assert gn(x=None) == 1 and gn(out=None) == 1 and gn(ws=None) == 1
    assert gn(B=-1) == 2 and gn(C=0) == 2 and gn(groups=0) == 2 and gn(groups=7) == 2 and gn(row=56) == 2 and gn(eps=-1.0) == 2
    assert gn(eps=float("nan")) == 2 and gn(C=8200, row=8200, orow=8200) == 2 and gn(B=65536) == 2
    assert gn(C=60, groups=4) == 3 and gn(row=68) == 3 and gn(batch=257) == 3 and gn(x=p + 8) == 3 and gn(out=p + 2) == 3 and gn(ws=p + 4) == 3
    assert gn(w=p + 2) == 3 and gn(b=p + 8, f32=1) == 3
    assert gn(dtype=2) == 4 and gn(act=2) == 7 and gn(wsb=0) == 8

    def q8(C=64, z=None, q=p, s=p, x=p):
        return lib.pq_group_norm_quant_rows(x, 0, 1, 4, C, C, 4 * C, 8, None, None, 0, 1e-6, 0, z, C, 4 * C, q, s, p, big, None, None)
    assert q8(q=None) == 1 and q8(s=None) == 1 and q8(C=72) == 3 and q8(q=p + 8) == 3 and q8(z=p + 8) == 3 and q8(x=None) == 1

    def q4(C=64, fmt=1, codes=p, scales=p, row=p):
        return lib.pq_group_norm_quant_fp4(p, 0, 1, 4, C, C, 4 * C, 8, None, None, 0, 1e-6, 0, fmt, codes, scales, row, p, big, None, None)
    assert q4(fmt=2) == 7 and q4(codes=None) == 1 and q4(scales=None) == 1 and q4(row=None) == 1 and q4(C=80) == 3 and q4(scales=p + 4) == 3
    assert lib.pq_group_norm_workspace_bytes(1, 4, 64, 8) >= 64 and lib.pq_group_norm_workspace_bytes(0, 4, 64, 8) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("affine", ["as_x", "fp32"])
def test_silu_of_every_value(cuda_dev, dtype, affine):
    """A weight of zero leaves z = bias exactly: SiLU of every value of the type, tails, subnormals, infinities and NaN among them,
    beside partners of every size.  The bound is that of the activation above, then the rounding to 16 bits.  Below z = -41.5, -infinity
    included (its limit is 0), SiLU is between -41.5 / (1 + e^41.5) = -3.95e-17 and 0, and one such value may stand for all of them:
    off by at most 4e-17."""
    bits = torch.arange(-32768, 32768, dtype=torch.int32).to(torch.int16)
    v = bits.view(dtype)
    order = torch.randperm(v.numel(), generator=torch.Generator().manual_seed(1))
    x = torch.randn(2, 3, 8192, generator=torch.Generator().manual_seed(2)).to(dtype).to(cuda_dev)
    t = dtype if affine == "as_x" else torch.float32
    weight = torch.zeros(8192, dtype=t, device=cuda_dev)
    fi = torch.finfo(dtype)
    for values in (v, v[order]):
        for b in values.to(t).reshape(8, 8192):
            z = b.double()
            want = torch.where(z == -float("inf"), 0.0, z / (1 + torch.exp(-z)))
            got = norm_exec.group_norm_rows(x, 32, weight, b.to(cuda_dev), 1e-6, "silu").cpu().double()
            assert torch.equal(torch.isnan(got), torch.isnan(want).expand_as(got)), "NaN where the formula has it, and nowhere else"
            inf = torch.isinf(want)
            assert bool((got[..., inf] == want[inf]).all())
            ok = torch.isfinite(want)
            err = torch.where(z < -41.5, 4e-17, (11 + z.abs()) * 2.0 ** -24 * want.abs())
            bound = err + (want.abs() + err) * fi.eps / 2 + fi.smallest_normal * fi.eps / 2
            off = ((got - want).abs() / bound)[..., ok]
            assert float(off.max()) <= 1, (float(off.max()), z[ok][off.amax(dim=(0, 1)).argmax()])


@pytest.mark.gpu
def test_silu_far_below_zero(cuda_dev):
    """fp32 biases outside the 16-bit types' ranges: SiLU stays within 4e-17 of zero."""
    b = -torch.logspace(0, 38, 64)
    x = torch.randn(1, 4, 64, generator=torch.Generator().manual_seed(3)).bfloat16().to(cuda_dev)
    got = norm_exec.group_norm_rows(x, 8, torch.zeros(64, device=cuda_dev), b.to(cuda_dev), 1e-6, "silu")
    z = b.double()
    want = z / (1 + torch.exp(-z))
    assert bool((got.cpu().double() - want).abs().le(want.abs() * ((11 + z.abs()) * 2.0 ** -24 + 2.0 ** -8) + 4e-17).all())
    for rows in norm_exec.group_norm_quant_rows(x, 8, torch.zeros(64, device=cuda_dev), b.to(cuda_dev), 1e-6, "silu", want_normed=True)[2]:
        assert torch.equal(rows, got[0])


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["mx", "nv"])
@pytest.mark.parametrize("C,groups", [(32, 4), (96, 4), (224, 4), (320, 32), (672, 32)])
def test_scale_bytes_past_the_row(cuda_dev, fmt, C, groups):
    """The fused form writes every scale byte of its rows, the zeros behind a row's last scale among them, into memory that held
    others; products at those widths take its rows as they take the quantiser's."""
    x, w, b = (t.to(cuda_dev) for t in rows(2, 77, C, torch.bfloat16, C))
    z = norm_exec.group_norm_rows(x, groups, w, b, 1e-6, "silu").reshape(-1, C)
    shape = ops.fp4_scale_shape(154, C, fmt)
    assert ops.group_norm_quant_fp4_fused(x, groups, w, b, 1e-6, "silu", fmt) is not None

    def poisoned(call):
        del_me = [torch.full(shape, 255, dtype=torch.uint8, device=cuda_dev) for _ in range(8)]
        del del_me
        return call()
    f0 = poisoned(lambda: fp4_exec.quant_rows_fp4(z, fmt))
    f = poisoned(lambda: norm_exec.group_norm_quant_fp4(x, groups, w, b, 1e-6, "silu", fmt))
    r = torch.arange(154, device=cuda_dev)
    for tile in range(shape[1]):
        for k in range(4):
            at = (r % 32) * 16 + (r // 32 % 4) * 4 + k
            assert torch.equal(f.scales[r // 128, tile, at], f0.scales[r // 128, tile, at])
            if tile * 4 + k >= C // ops.FP4_BLOCK[fmt]:
                assert not f.scales[r // 128, tile, at].any()
    wq = fp4_exec.quant_rows_fp4(torch.randn(72, C, generator=torch.Generator().manual_seed(1)).bfloat16().to(cuda_dev), fmt)
    y = fp4_exec.fp4_gemm(f, wq)
    assert bool(torch.isfinite(y).all()) and torch.equal(y, fp4_exec.fp4_gemm(f0, wq))
