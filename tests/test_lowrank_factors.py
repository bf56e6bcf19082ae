"""Low-rank branches follow their factors: replaced, moved or edited ones, in eager calls and in replayed graphs."""
import ctypes

import pytest
import torch
import torch.nn as nn

from pyraquant_b200 import _lib, fp4_exec, int8_exec, ops

FMTS = ["mx", "nv"]
DTYPES = [torch.bfloat16, torch.float16]


def layer(cls, dev, K=640, N=328, dtype=torch.bfloat16, seed=4, **kw):
    g = torch.Generator().manual_seed(seed)
    lin = nn.Linear(K, N).to(dtype)
    with torch.no_grad():
        lin.weight.copy_(torch.randn(N, K, generator=g) / K ** 0.5)
        lin.bias.copy_(torch.randn(N, generator=g))
    A, B = torch.randn(K, 32, generator=g) / K ** 0.5, torch.randn(32, N, generator=g) / 5
    return cls(lin, device=dev, lowrank=(A.to(dtype), B.to(dtype)), **kw)


def by_parts(m, x):
    """The layer's steps one by one, the up-projection laid out on the spot."""
    xq = fp4_exec.quant_rows_fp4(x, m.fmt)
    factors = fp4_exec.lowrank_rows(m._down(x), xq), fp4_exec.lowrank_weight(m.lr_B, m.weight_rows)
    return fp4_exec.fp4_gemm(xq, m.weight_rows, m.bias, x.dtype, factors)


# ------------------------------------------------------------------------------------------------ the two factors in one launch
@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("t_type", DTYPES)
@pytest.mark.parametrize("b_type", DTYPES)
def test_factors_are_laid_out_as_their_parts_are(cuda_dev, fmt, t_type, b_type, monkeypatch):
    g = torch.Generator().manual_seed(3)
    for M, N in ((1, 1), (63, 64), (64, 65), (300, 1280), (0, 40), (5, 10240)):
        xq = fp4_exec.quant_rows_fp4((torch.randn(M, 32, generator=g) * 50).to(t_type).to(cuda_dev), fmt)
        w = fp4_exec.quant_rows_fp4(torch.randn(N, 32, generator=g).bfloat16().to(cuda_dev), fmt)
        t, B = torch.randn(M, 32, generator=g).to(t_type).to(cuda_dev), torch.randn(32, N, generator=g).to(b_type).to(cuda_dev)
        want = fp4_exec.lowrank_rows(t, xq), fp4_exec.lowrank_weight(B, w)
        got = fp4_exec.lowrank_factors(t, xq, B, w)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]) and got[1].is_contiguous()
        wide = torch.zeros(32, N + 3, dtype=b_type, device=cuda_dev)
        wide[:, 3:] = B
        off = torch.zeros(M, 40, dtype=t_type, device=cuda_dev)
        off[:, 3:35] = t
        got = fp4_exec.lowrank_factors(off[:, 3:35], xq, wide[:, 3:], w)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    lib = _lib.load()                                             # rows of B that lie apart, nothing else written
    out = torch.full((70 * 32 + 8,), 7.0, device=cuda_dev)
    B = torch.randn(32, 91, generator=g).to(b_type).to(cuda_dev)
    assert lib.pq_fp4_lowrank_factors(None, 0, None, None, 0, B.data_ptr() + 2 * 5, ops._DT[b_type], 91, None, out.data_ptr(), 70,
                                      torch.cuda.current_stream().cuda_stream) == 0
    assert torch.equal(out[: 70 * 32].reshape(70, 32), B[:, 5:75].t().float()) and bool((out[70 * 32:] == 7).all())


@pytest.mark.gpu
def test_factors_refusals(cuda_dev):
    x = torch.randn(9, 96, device=cuda_dev).bfloat16()
    xq, w = fp4_exec.quant_rows_fp4(x, "nv"), fp4_exec.quant_rows_fp4(torch.randn(40, 96, device=cuda_dev).bfloat16(), "nv")
    t, B = torch.randn(9, 32, device=cuda_dev).bfloat16(), torch.randn(32, 40, device=cuda_dev).bfloat16()
    for bad in ((t[:, :16], xq, B, w), (t, xq, B[:, :39], w), (t, xq, B[:16], w), (t[:8], xq, B, w), (t, xq, B.cpu(), w), (t.cpu(), xq, B, w),
                (t[None], xq, B, w), (t, fp4_exec.Fp4Rows(xq.codes, xq.scales, xq.row_scale.double()), B, w)):
        with pytest.raises(AssertionError):
            fp4_exec.lowrank_factors(*bad)
    for bad in ((t.float(), xq, B, w), (t, xq, B.float(), w)):
        with pytest.raises(TypeError):
            fp4_exec.lowrank_factors(*bad)


@pytest.mark.gpu
def test_layout_general_path_agrees_with_the_one_step_call(cuda_dev, monkeypatch):
    A, B = torch.randn(90, 32, device=cuda_dev).half(), torch.randn(32, 70, device=cuda_dev).bfloat16()
    t, x = torch.randn(9, 32, device=cuda_dev).half(), fp4_exec.quant_rows_fp4(torch.randn(9, 32, device=cuda_dev).half(), "nv")
    w = fp4_exec.quant_rows_fp4(torch.randn(70, 32, device=cuda_dev).half(), "nv")
    bind = ops._BIND()
    for good in ((A, B), (A, None), (None, B)):
        assert bind.lowrank_layout(*good) is not None
    for bad in ((A.float(), B), (A[:, :16], None), (A.cpu(), B), (None, B[:31]), (None, None), ("A", B), (A.t().contiguous().t(), B)):
        assert bind.lowrank_layout(*bad) is None
    assert bind.fp4_lowrank_factors(t, x.row_scale, B, w.row_scale) is not None
    for bad in ((t, None, B[:, ::2], None), (t, w.row_scale, B, None), (t, None, B, x.row_scale), (t.float(), None, B, None), (t, None, B, "c"), (t, None, None, None)):
        assert bind.fp4_lowrank_factors(*bad) is None
    one = (*ops.lowrank_layout(A, B), *fp4_exec.lowrank_factors(t, x, B, w))

    class Refuses:
        def __getattr__(self, name):
            return lambda *a: None
    monkeypatch.setattr(ops, "_bind_handle", Refuses())
    assert all(torch.equal(a, b) for a, b in zip(one, (*ops.lowrank_layout(A, B), *fp4_exec.lowrank_factors(t, x, B, w))))


def test_factors_argument_checks():
    lib = _lib.load()
    buf = ctypes.create_string_buffer(4096)
    p = (ctypes.addressof(buf) + 63) & ~63

    def f(t=p, td=0, row=p, t_out=p, M=4, b=p, bd=0, ldb=8, col=p, b_out=p, N=8):
        return lib.pq_fp4_lowrank_factors(t, td, row, t_out, M, b, bd, ldb, col, b_out, N, None)
    assert f(M=0, N=0, t=None, b=None) == 0
    assert f(M=-1) == 2 and f(N=-1) == 2 and f(ldb=7) == 2 and f(M=1 << 40) == 2 and f(N=1 << 40) == 2
    assert f(td=2) == 4 and f(bd=2) == 4
    assert f(t=None) == 1 and f(t_out=None) == 1 and f(b=None) == 1 and f(b_out=None) == 1
    assert f(t=p + 8) == 3 and f(t_out=p + 16) == 3 and f(b=p + 1) == 3 and f(b_out=p + 16) == 3 and f(row=p + 2) == 3 and f(col=p + 2) == 3


# ------------------------------------------------------------------------------------------------ Fp4Linear: the up-projection
@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FMTS)
def test_fp4_follows_a_replaced_up_projection(cuda_dev, fmt):
    """A factor taken off before its successor is made, which the allocator puts where the old one was; a round trip over the
    CPU with an edit; a write that torch does not count."""
    m = layer(fp4_exec.Fp4Linear, cuda_dev, fmt=fmt)
    x = torch.randn(75, 640, device=cuda_dev).bfloat16()
    m(x)
    same = 0
    for i in range(20):
        before = m.lr_B.data_ptr()
        m.lr_B = None
        m.lr_B = torch.randn(32, 328, device=cuda_dev, dtype=torch.bfloat16)
        same += m.lr_B.data_ptr() == before
        assert torch.equal(m(x), by_parts(m, x)), i
    assert same > 0                                               # or the test shows nothing
    m.cpu()
    m.lr_B.mul_(3)
    m.cuda()
    assert torch.equal(m(x), by_parts(m, x))
    m.lr_B.data.mul_(-2)
    assert torch.equal(m(x), by_parts(m, x))


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FMTS)
def test_fp4_graph_follows_the_up_projection(cuda_dev, fmt):
    """A layer that ran before the capture: replays use the factor as it is then, whatever eager calls ran in between."""
    m = layer(fp4_exec.Fp4Linear, cuda_dev, fmt=fmt)
    x = torch.randn(75, 640, device=cuda_dev).bfloat16()
    m(x)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = m(x)
    graph.replay()
    assert torch.equal(y, by_parts(m, x))
    m.lr_B.mul_(-2)
    graph.replay()
    assert torch.equal(y, by_parts(m, x))
    m(x)
    filler = [torch.full((328, 32), 1e4, device=cuda_dev) for _ in range(8)]
    graph.replay()
    assert torch.equal(y, by_parts(m, x))
    del filler
    ops.check_device_status(cuda_dev)


# ------------------------------------------------------------------------------------------------ both Linears: the kept copies
LAYERS = [(int8_exec.Int8Linear, {}), (fp4_exec.Fp4Linear, {"fmt": "mx"}), (fp4_exec.Fp4Linear, {"fmt": "nv"})]
layers = pytest.mark.parametrize("cls,kw", LAYERS, ids=["int8", "fp4_mx", "fp4_nv"])
factors = pytest.mark.parametrize("name", ["lr_A", "lr_B"])


def by_fresh_layer(m, x, **kw):
    """What a layer with these factors that has never run gives."""
    n = layer(type(m), x.device, **kw)
    n.lr_A, n.lr_B = m.lr_A.clone(), m.lr_B.clone()
    return n(x)


def transposed(m, name):
    return m._lr_At() if name == "lr_A" else m._lr_Bt()


@factors
def test_transposed_copies_follow_replacements(name):
    m = layer(int8_exec.Int8Linear, torch.device("cpu"))
    shape, dtype = getattr(m, name).shape, getattr(m, name).dtype
    for i in range(100):                                          # the allocator often hands the same place out again
        setattr(m, name, None)
        setattr(m, name, torch.randn(shape).to(dtype))
        assert torch.equal(transposed(m, name), getattr(m, name).t()), i
    kept = transposed(m, name)
    assert transposed(m, name) is kept                            # laid out once
    getattr(m, name).mul_(2)
    assert torch.equal(transposed(m, name), getattr(m, name).t())
    m.half()
    assert torch.equal(transposed(m, name), getattr(m, name).t()) and transposed(m, name).dtype == torch.float16
    getattr(m, name).data = torch.randn(shape).half()
    assert torch.equal(transposed(m, name), getattr(m, name).t())


@factors
def test_transposed_copies_in_inference_mode(name):
    """Inference tensors count no writes: their copies are made anew.  Ordinary factors written inside inference mode are followed."""
    with torch.inference_mode():
        m = layer(int8_exec.Int8Linear, torch.device("cpu"))
        transposed(m, name)
        getattr(m, name).mul_(2)
        assert torch.equal(transposed(m, name), getattr(m, name).t())
    getattr(m, name)
    assert torch.equal(transposed(m, name), getattr(m, name).t())
    m = layer(int8_exec.Int8Linear, torch.device("cpu"))
    transposed(m, name)
    with torch.inference_mode():
        getattr(m, name).mul_(2)
        assert torch.equal(transposed(m, name), getattr(m, name).t())
    assert torch.equal(transposed(m, name), getattr(m, name).t())


@pytest.mark.gpu
@layers
@factors
def test_layers_follow_their_factors(cuda_dev, cls, kw, name):
    m = layer(cls, cuda_dev, **kw)
    x = torch.randn(75, 640, device=cuda_dev).bfloat16()
    m(x)
    shape = getattr(m, name).shape
    for i in range(10):
        setattr(m, name, None)
        setattr(m, name, torch.randn(shape, device=cuda_dev, dtype=torch.bfloat16))
        assert torch.equal(m(x), by_fresh_layer(m, x, **kw)), i
    getattr(m, name).mul_(2)
    assert torch.equal(m(x), by_fresh_layer(m, x, **kw))
    m.cpu()
    getattr(m, name).mul_(-2)
    m.cuda()
    assert torch.equal(m(x), by_fresh_layer(m, x, **kw))
    if cls is fp4_exec.Fp4Linear:                                 # keeps nothing: not even a write that torch does not count is missed
        getattr(m, name).data.mul_(-2)
        assert torch.equal(m(x), by_fresh_layer(m, x, **kw))
        assert not [k for k, v in m.__dict__.items() if k.startswith("_t_cache")]
    with torch.inference_mode():
        n = layer(cls, cuda_dev, **kw)
        n(x)
        getattr(n, name).mul_(2)
        got = n(x)
        assert torch.equal(got, by_fresh_layer(n, x, **kw))


@pytest.mark.gpu
@layers
@factors
@pytest.mark.parametrize("warm", [True, False])
def test_graphs_follow_the_factors(cuda_dev, cls, kw, name, warm):
    """Replays use the factors as they are then, whether the layer ran before the capture or not, and whatever ran in between."""
    layer(cls, cuda_dev, **kw)(torch.randn(75, 640, device=cuda_dev).bfloat16())           # libraries and kernels are loaded
    m = layer(cls, cuda_dev, **kw)
    x = torch.randn(75, 640, device=cuda_dev).bfloat16()
    if warm:
        m(x)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = m(x)
    eager = m(x)                                                  # before anything of the capture has run
    assert torch.equal(eager, by_fresh_layer(m, x, **kw))
    graph.replay()
    assert torch.equal(y, eager)
    getattr(m, name).mul_(-2)
    graph.replay()
    assert torch.equal(y, by_fresh_layer(m, x, **kw))
    m(x)
    filler = [torch.full((640, 32), 1e4, device=cuda_dev, dtype=torch.bfloat16) for _ in range(8)]
    graph.replay()
    assert torch.equal(y, by_fresh_layer(m, x, **kw))
    del filler
    ops.check_device_status(cuda_dev)


@pytest.mark.gpu
@layers
def test_first_call_on_another_stream(cuda_dev, cls, kw):
    """A copy that one stream is still to make is waited for by a call on another one, and lives until that call has read it."""
    layer(cls, cuda_dev, **kw)(torch.randn(75, 640, device=cuda_dev).bfloat16())
    side = torch.cuda.Stream()
    x = torch.randn(75, 640, device=cuda_dev).bfloat16()
    for i in range(5):
        m = layer(cls, cuda_dev, **kw, seed=10 + i)
        want = by_fresh_layer(m, x, **kw, seed=10 + i)
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            torch.cuda._sleep(20_000_000)                         # some 10 ms
            first = m(x)
        here = m(x)
        assert torch.equal(here, want)
        torch.cuda.synchronize()
        assert torch.equal(first, want)
    torch.cuda.synchronize()
    m = layer(cls, cuda_dev, **kw)
    want = by_fresh_layer(m, x, **kw)
    m(x)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        torch.cuda._sleep(20_000_000)
        late = m(x)
    old = m.lr_A, m.lr_B                                          # the factors stay for the call that is still to read them
    m.lr_A, m.lr_B = m.lr_A.clone(), m.lr_B.clone()               # here: the copies go, and their memory is written again
    m(x)
    filler = [torch.full((640 * 32,), 1e4, device=cuda_dev, dtype=torch.bfloat16) for _ in range(64)]
    torch.cuda.synchronize()
    assert torch.equal(late, want)
    del filler, old


@layers
def test_kept_copies_stay_with_the_layer(cls, kw):
    """Pickles and copies hold the buffers alone, a layer that is converted or moved drops what it kept."""
    import copy
    import pickle
    m = layer(cls, torch.device("cpu"), **kw)
    size = len(pickle.dumps(m))
    before = set(m.__dict__)
    m._lr_At(), m._lr_Bt()
    assert len(pickle.dumps(m)) == size
    for n in (pickle.loads(pickle.dumps(m)), copy.deepcopy(m), copy.copy(m)):
        assert set(n.__dict__) == before and torch.equal(n.lr_A, m.lr_A) and torch.equal(n._lr_At(), m._lr_At())
    assert set(m.half().__dict__) == before


@pytest.mark.gpu
@layers
def test_a_layer_moved_off_leaves_no_memory(cuda_dev, cls, kw):
    x = torch.randn(75, 640, device=cuda_dev).bfloat16()
    layer(cls, cuda_dev, **kw)(x)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated(cuda_dev)
    m = layer(cls, cuda_dev, **kw)
    m(x)
    m.cpu()
    torch.cuda.synchronize()
    assert torch.cuda.memory_allocated(cuda_dev) == before


# ------------------------------------------------------------------------------------------------ the copies of a graph
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_layout_of_both_factors(cuda_dev, dtype):
    g = torch.Generator().manual_seed(5)
    for K, N in ((1, 1), (63, 64), (65, 129), (640, 328), (10240, 7), (7, 10240)):
        A, B = torch.randn(K, 32, generator=g).to(dtype).to(cuda_dev), torch.randn(32, N, generator=g).to(dtype).to(cuda_dev)
        for a, b in ((A, B), (A, None), (None, B)):
            at, bt = ops.lowrank_layout(a, b)
            assert at is None if a is None else (torch.equal(at, A.t()) and at.is_contiguous())
            assert bt is None if b is None else (torch.equal(bt, B.t()) and bt.is_contiguous())
    wide = torch.randn(70, 40, generator=g).to(dtype).to(cuda_dev)
    for a, b in ((wide[:, 1:33], wide[:32, 3:]), (wide[:, :32].t().contiguous().t(), wide[:32]), (wide, wide[:16]), (wide.float()[:, :32].contiguous(), None)):
        at, bt = ops.lowrank_layout(a, b)                         # what the kernel does not take as it is
        assert torch.equal(at, a.t()) and at.is_contiguous() and (b is None or (torch.equal(bt, b.t()) and bt.is_contiguous()))
    lib, A = _lib.load(), torch.randn(9, 48, generator=g).to(dtype).to(cuda_dev)
    out = torch.full((32 * 9 + 8,), 7.0, dtype=dtype, device=cuda_dev)            # rows apart, nothing else written
    assert lib.pq_lowrank_layout(A.data_ptr() + 16, 48, out.data_ptr() + 2, 9, None, 0, None, 0, torch.cuda.current_stream().cuda_stream) == 0
    assert torch.equal(out[1: 289].reshape(32, 9), A[:, 8:40].t()) and bool((out[289:] == 7).all()) and float(out[0]) == 7


def test_layout_argument_checks():
    lib = _lib.load()
    buf = ctypes.create_string_buffer(4096)
    p = (ctypes.addressof(buf) + 63) & ~63

    def f(a=p, lda=32, a_t=p, K=4, b=p, ldb=8, b_t=p, N=8):
        return lib.pq_lowrank_layout(a, lda, a_t, K, b, ldb, b_t, N, None)
    assert f(K=0, N=0, a=None, b=None) == 0
    assert f(K=-1) == 2 and f(N=-1) == 2 and f(lda=24) == 2 and f(ldb=7) == 2 and f(K=1 << 31) == 2
    assert f(a=None) == 1 and f(a_t=None) == 1 and f(b=None) == 1 and f(b_t=None) == 1
    assert f(lda=36) == 3 and f(a=p + 8) == 3 and f(a_t=p + 1) == 3 and f(b=p + 1) == 3 and f(b_t=p + 8) == 3


# ------------------------------------------------------------------------------------------------ torch.compile
@pytest.mark.gpu
@layers
@pytest.mark.parametrize("norm", [False, True])
def test_compiled_layers_give_the_eager_values(cuda_dev, cls, kw, norm):
    """``torch.compile`` of a layer's forward and of its group-norm form, with a branch and without: the eager values, also after the
    factors were written in place and replaced."""
    torch._dynamo.reset()
    m = layer(cls, cuda_dev, **kw)
    plain = cls(nn.Linear(640, 328).bfloat16(), device=cuda_dev, **kw)
    x = torch.randn(2, 75, 640, device=cuda_dev).bfloat16()
    w = torch.randn(640, device=cuda_dev).bfloat16()

    def call(n, x):
        return n.forward_group_norm(x, 32, w, w, 1e-6, "silu") if norm else n(x)
    compiled = torch.compile(call, backend="aot_eager")
    with torch.no_grad():
        assert torch.equal(compiled(plain, x), call(plain, x))
        for i in range(6):
            # the compiled call may sum x @ A in another kernel: a rounding of t, then of y
            want = call(m, x)
            got = compiled(m, x)
            tol = 4 * torch.finfo(x.dtype).eps * float(want.abs().max())
            assert float((got.float() - want.float()).abs().max()) <= tol, i
            name = ("lr_A", "lr_B")[i % 2]
            if i < 2:
                getattr(m, name).mul_(-2)
            elif i < 4:
                setattr(m, name, torch.randn_like(getattr(m, name)) / 8)
            else:
                m.cpu()
                getattr(m, name).mul_(2)
                m.cuda()


def test_one_step_calls_leave_cpu_operands_alone():
    bind = _lib.binding()
    A, B = torch.randn(40, 32).bfloat16(), torch.randn(32, 24).bfloat16()
    assert bind.lowrank_layout(A, B) is None and bind.lowrank_layout(None, None) is None and bind.lowrank_layout(A) is None and bind.lowrank_layout(3, B) is None
    assert bind.fp4_lowrank_factors(A, None, B, None) is None and bind.fp4_lowrank_factors(A, None, "B", None) is None and bind.fp4_lowrank_factors() is None
    at, bt = ops.lowrank_layout(A, B)
    assert torch.equal(at, A.t()) and torch.equal(bt, B.t()) and at.is_contiguous() and bt.is_contiguous()
    q = fp4_exec.quantize_weight_fp4(torch.randn(40, 32))
    w = fp4_exec.quantize_weight_fp4(torch.randn(24, 32))
    with pytest.raises(AssertionError):
        fp4_exec.lowrank_factors(A, q, B, w)
