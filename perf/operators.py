"""Cases of the 4-bit floating-point Linear and of the group norm in front of it: quantisation and reading back, the
product, the norm, and norm + quantisation + product as a projection behind a group norm runs them.

A case's `op` says which operator:
  quant        rows of 16-bit activations -> packed 4-bit rows -> the values that these stand for
  product      packed activations x packed weights (+ bias) -> 16-bit rows
  norm         group norm (and SiLU) over channels-last rows
  norm_linear  group norm whose output is quantised to 4 bits, then the product with a packed weight
`own` selects between the plain form (elementary torch operations in 32 bits) and the package's operators.

Formats (`fmt`): "mx" has one power-of-two scale (E8M0) per 32 elements; "nv" one E4M3 scale per 16 elements and a
power of two per row above it.  Elements are E2M1 codes, two per byte, the even one in the low nibble.  Scale bytes stand
in tiles of 128 rows x 4 scales: [row tile, scale tile, row % 32, row // 32 % 4, scale % 4].
"""
import torch

own = False

BLOCK = {"mx": 32, "nv": 16}
DTYPE = {"bf16": torch.bfloat16, "fp16": torch.float16}
GROUPS, EPS = 32, 1e-6


def listed():
    return [
        # one token's activations in front of a Linear: nothing but latency
        {"name": "quant_nv_1x5120", "op": "quant", "fmt": "nv", "dtype": "bf16", "M": 1, "K": 5120},
        # a ragged batch of image tokens in front of a 640-channel projection
        {"name": "quant_mx_4173x640", "op": "quant", "fmt": "mx", "dtype": "fp16", "M": 4173, "K": 640},
        # the feed-forward's second Linear over all tokens of a high-resolution batch
        {"name": "quant_nv_16384x5120", "op": "quant", "fmt": "nv", "dtype": "bf16", "M": 16384, "K": 5120},
        # one token through the feed-forward's first Linear: the weights are read for a single row
        {"name": "product_nv_1x1280x10240", "op": "product", "fmt": "nv", "dtype": "bf16", "M": 1, "K": 1280, "N": 10240, "bias": True},
        # the 77 text tokens through a cross-attention projection
        {"name": "product_mx_77x2048x1280", "op": "product", "fmt": "mx", "dtype": "fp16", "M": 77, "K": 2048, "N": 1280, "bias": False},
        # the feed-forward's first Linear over all tokens
        {"name": "product_nv_16384x1280x10240", "op": "product", "fmt": "nv", "dtype": "bf16", "M": 16384, "K": 1280, "N": 10240, "bias": True},
        # a large square product: the tensor cores' own rate
        {"name": "product_mx_8192x8192x8192", "op": "product", "fmt": "mx", "dtype": "bf16", "M": 8192, "K": 8192, "N": 8192, "bias": False},
        # the norm of the innermost blocks, 32 x 32 positions
        {"name": "norm_1x1024x1280", "op": "norm", "dtype": "fp16", "B": 1, "T": 1024, "C": 1280, "silu": True},
        # the norm of the outermost blocks, 128 x 128 positions, two images
        {"name": "norm_2x16384x320", "op": "norm", "dtype": "bf16", "B": 2, "T": 16384, "C": 320, "silu": True},
        # the norm of an image decoder's blocks at 512 x 512: far more than the chip holds
        {"name": "norm_1x262144x256", "op": "norm", "dtype": "bf16", "B": 1, "T": 262144, "C": 256, "silu": True},
        # norm and projection in front of a block's attention, a ragged image
        {"name": "norm_linear_3x2491x640", "op": "norm_linear", "fmt": "mx", "dtype": "fp16", "B": 3, "T": 2491, "C": 640, "N": 640, "bias": True, "silu": False},
        # the same at 64 x 64, two images
        {"name": "norm_linear_2x4096x640", "op": "norm_linear", "fmt": "nv", "dtype": "bf16", "B": 2, "T": 4096, "C": 640, "N": 640, "bias": True, "silu": False},
    ]


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    op = rng.choice(["quant", "product", "product", "norm", "norm_linear"])
    case = {"op": op, "dtype": rng.choice(["bf16", "fp16"])}
    if op == "quant":
        K = 32 * _log(rng, 1, 320)
        return dict(case, fmt=rng.choice(["mx", "nv"]), M=_log(rng, 1, min(16384, 16384 * 5120 // K)), K=K)
    if op == "product":
        K, N = 32 * _log(rng, 1, 256), _log(rng, 8, 10240)
        return dict(case, fmt=rng.choice(["mx", "nv"]), M=_log(rng, 1, min(16384, 8192 ** 3 // (K * N))), K=K, N=N, bias=rng.random() < 0.5)
    C = 32 * _log(rng, 1, 60)
    B = rng.randint(1, 4)
    most = 262144 * 256 // (B * C) if op == "norm" else 8192 * 640 // (B * C)
    case.update(B=B, T=_log(rng, 1, most), C=C, silu=rng.random() < 0.5)
    if op == "norm_linear":
        case.update(fmt=rng.choice(["mx", "nv"]), N=_log(rng, 8, 2560), bias=rng.random() < 0.5)
    return case


def _rows(case, rows, cols, g):
    """16-bit activations: normal, with one channel in 200 twenty times as large."""
    x = torch.randn(rows, cols, generator=g, device="cuda")
    far = torch.randperm(cols, generator=g, device="cuda")[: max(1, cols // 200)]
    x[:, far] *= 20.0
    return x.to(DTYPE[case["dtype"]])


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    state = {"case": dict(case)}
    if case["op"] == "quant":
        state["x"] = _rows(case, case["M"], case["K"], g)
        return state
    if case["op"] == "product":
        state["x"] = _quantise(_rows(case, case["M"], case["K"], g), case["fmt"])
        K = case["K"]
    else:
        B, T, C = case["B"], case["T"], case["C"]
        t = DTYPE[case["dtype"]]
        x = torch.randn(B * T, C, generator=g, device="cuda") * (0.5 + torch.rand(C, generator=g, device="cuda"))
        state["x"] = (x + 0.5 * torch.randn(C, generator=g, device="cuda")).to(t).reshape(B, T, C)
        state["gamma"] = (1 + 0.2 * torch.randn(C, generator=g, device="cuda")).to(t)
        state["beta"] = (0.2 * torch.randn(C, generator=g, device="cuda")).to(t)
        K = C
    if "N" in case:
        w = torch.randn(case["N"], K, generator=g, device="cuda") / K ** 0.5
        state["w"] = _quantise(w.to(torch.bfloat16), case["fmt"])
        state["bias"] = 0.1 * torch.randn(case["N"], generator=g, device="cuda") if case["bias"] else None
    return state


# ------------------------------------------------------------------------------------------------ plain form
def _quantise(x, fmt):
    """(codes [M, K/2], tiled scale bytes, row scales [M] or None) of 16-bit rows."""
    M, K = x.shape
    b = x.float().reshape(M, K // BLOCK[fmt], BLOCK[fmt])
    amax = b.abs().amax(dim=2)
    row = None
    if fmt == "mx":
        # exponent of the block's largest magnitude, less the 2 of the largest E2M1 value
        byte = ((amax.view(torch.int32) >> 23) - 2).clamp(min=0)
        q = torch.ldexp(b, (127 - byte)[:, :, None])
        byte = byte.to(torch.uint8)
    else:
        m, e = torch.frexp(amax.amax(dim=1))                      # m in [0.5, 1): the row's largest is m * 2^e
        e = torch.where(m > 0.65625, e - 11, e - 12)              # smallest e with largest / (6 * 448) <= 2^e
        row = torch.ldexp(torch.ones_like(m), torch.where(m > 0, e, torch.zeros_like(e)).clamp(min=-100))
        s8 = (amax / row[:, None] / 6).to(torch.float8_e4m3fn)
        s = s8.float()[:, :, None]
        q = torch.where(s > 0, b / row[:, None, None] / torch.where(s > 0, s, torch.ones_like(s)), torch.zeros_like(b))
        byte = s8.view(torch.uint8)
    a = q.abs()
    code = ((a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5))
    code = (code + 8 * torch.signbit(b)).to(torch.uint8).reshape(M, K)
    codes = code[:, 0::2] | (code[:, 1::2] << 4)
    nb = K // BLOCK[fmt]
    tiled = torch.zeros((M + 127) // 128 * 128, (nb + 3) // 4 * 4, dtype=torch.uint8, device=x.device)
    tiled[:M, :nb] = byte
    tiled = tiled.reshape((M + 127) // 128, 4, 32, (nb + 3) // 4, 4).permute(0, 3, 2, 1, 4)
    return codes.contiguous(), tiled.reshape((M + 127) // 128, (nb + 3) // 4, 512).contiguous(), row


def _values(q, fmt):
    """fp32 values of packed rows."""
    codes, tiled, row = q
    M, K = codes.shape[0], codes.shape[1] * 2
    nb = K // BLOCK[fmt]
    byte = tiled.reshape(tiled.shape[0], tiled.shape[1], 32, 4, 4).permute(0, 3, 2, 1, 4).reshape(tiled.shape[0] * 128, -1)[:M, :nb]
    table = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], device=codes.device)
    table = torch.cat([table, -table])
    v = table[torch.stack([codes & 15, codes >> 4], dim=2).reshape(M, K).long()].reshape(M, nb, BLOCK[fmt])
    if fmt == "mx":
        s = torch.ldexp(torch.ones_like(byte, dtype=torch.float32), byte.int() - 127)
    else:
        s = byte.contiguous().view(torch.float8_e4m3fn).float() * row[:, None]
    return (v * s[:, :, None]).reshape(M, K)


def _round(v, t):
    return v.clamp(-65504, 65504).to(t) if t == torch.float16 else v.to(t)


def _norm(state):
    case, x = state["case"], state["x"].float()
    B, T, C = x.shape
    g = x.reshape(B, T, GROUPS, C // GROUPS)
    mean = g.mean(dim=(1, 3), keepdim=True)
    g = g - mean
    g = g * torch.rsqrt((g * g).mean(dim=(1, 3), keepdim=True) + EPS)
    z = g.reshape(B, T, C) * state["gamma"].float() + state["beta"].float()
    return (z * torch.sigmoid(z) if case["silu"] else z).to(DTYPE[case["dtype"]])


def _product(xq, wq, bias, fmt, t):
    y = _values(xq, fmt) @ _values(wq, fmt).t()
    return (y + bias if bias is not None else y).to(t)


def run(state):
    case = state["case"]
    op, t = case["op"], DTYPE[case["dtype"]]
    if own:
        from pyraquant_b200 import fp4_exec, norm_exec
        if op == "quant":
            return fp4_exec.dequant_rows_fp4(fp4_exec.quant_rows_fp4(state["x"], case["fmt"]), t)
        if op == "product":
            return fp4_exec.fp4_gemm(fp4_exec.Fp4Rows(*state["x"]), fp4_exec.Fp4Rows(*state["w"]), state["bias"], t)
        act = "silu" if case["silu"] else None
        if op == "norm":
            return norm_exec.group_norm_rows(state["x"], GROUPS, state["gamma"], state["beta"], EPS, act)
        xq = norm_exec.group_norm_quant_fp4(state["x"], GROUPS, state["gamma"], state["beta"], EPS, act, case["fmt"])
        return fp4_exec.fp4_gemm(xq, fp4_exec.Fp4Rows(*state["w"]), state["bias"], t)
    if op == "quant":
        return _round(_values(_quantise(state["x"], case["fmt"]), case["fmt"]), t)
    if op == "product":
        return _product(state["x"], state["w"], state["bias"], case["fmt"], t)
    z = _norm(state)
    if op == "norm":
        return z
    return _product(_quantise(z.reshape(-1, case["C"]), case["fmt"]), state["w"], state["bias"], case["fmt"], t)


def _packed_bytes(rows, K, fmt):
    return rows * (K // 2 + K // BLOCK[fmt] + (4 if fmt == "nv" else 0))


def work(case):
    op = case["op"]
    if op == "quant":
        M, K = case["M"], case["K"]
        return {"bytes": 4 * M * K + _packed_bytes(M, K, case["fmt"]), "flops": 4 * M * K}
    if op == "product":
        M, N, K = case["M"], case["N"], case["K"]
        return {"bytes": _packed_bytes(M + N, K, case["fmt"]) + 2 * M * N + (4 * N if case["bias"] else 0), "flops": 2 * M * N * K}
    n = case["B"] * case["T"] * case["C"]
    if op == "norm":
        return {"bytes": 4 * n, "flops": 10 * n}
    N, rows = case["N"], case["B"] * case["T"]
    return {"bytes": 2 * n + _packed_bytes(N, case["C"], case["fmt"]) + 2 * rows * N + (4 * N if case["bias"] else 0),
            "flops": 10 * n + 2 * n * N}


# ------------------------------------------------------------------------------------------------ the definition in 64 bits
def _nearest(v, grid):
    """Index of the nearest value of an ascending grid, a tie going to the even index; past the end the last one."""
    hi = torch.searchsorted(grid, v.contiguous()).clamp(max=len(grid) - 1)
    lo = (hi - 1).clamp(min=0)
    below, above = v - grid[lo], grid[hi] - v
    return torch.where((below < above) | ((below == above) & (lo % 2 == 0)), lo, hi)


def _exact_quantised(x, fmt):
    """The values that quantised rows stand for, in 64 bits."""
    M, K = x.shape
    e2m1 = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64, device=x.device)
    b = x.double().reshape(M, -1, BLOCK[fmt])
    largest = b.abs().amax(dim=2)
    if fmt == "mx":
        s = torch.ldexp(torch.ones_like(largest), (torch.frexp(largest)[1] - 3).clamp(min=-127))
    else:
        per_row = largest.amax(dim=1) / (6 * 448)
        m, e = torch.frexp(per_row)
        e = torch.where(m == 0.5, e - 1, e)
        row = torch.ldexp(torch.ones_like(m), torch.where(per_row > 0, e, torch.zeros_like(e)).clamp(min=-100))
        k = torch.arange(127, device=x.device)
        e4m3 = torch.where(k < 8, k * 2.0 ** -9, torch.ldexp(1 + (k % 8).double() / 8, k // 8 - 7)).double()
        s = e4m3[_nearest(largest / row[:, None] / 6, e4m3)] * row[:, None]
    s = s[:, :, None]
    q = torch.where(s > 0, b.abs() / torch.where(s > 0, s, torch.ones_like(s)), torch.zeros_like(b))
    return (torch.sign(b) * e2m1[_nearest(q, e2m1)] * s).reshape(M, K)


def _exact_packed(q, fmt):
    """64-bit values of packed rows, byte by byte from the layout."""
    codes, tiled, row = q
    M, K = codes.shape[0], 2 * codes.shape[1]
    k = torch.arange(K, device=codes.device)
    code = (codes.long()[:, k // 2] >> (4 * (k % 2))) & 15
    mant, ex = code & 1, (code >> 1) & 3
    v = torch.where(ex == 0, mant * 0.5, (1 + mant.double() / 2) * torch.ldexp(torch.ones_like(ex, dtype=torch.float64), ex - 1))
    v = torch.where(code >= 8, -v, v)
    blk = (k // BLOCK[fmt])[None, :]
    r = torch.arange(M, device=codes.device)[:, None]
    byte = tiled.long()[r // 128, blk // 4, (r % 32) * 16 + (r // 32 % 4) * 4 + blk % 4]
    if fmt == "mx":
        return v * torch.ldexp(torch.ones_like(v), byte - 127)
    m, e = byte & 7, byte >> 3
    s = torch.where(e == 0, m * 2.0 ** -9, torch.ldexp(1 + m.double() / 8, e - 7))
    return v * s * row.double()[:, None]


def exact(case, seed):
    state = prepare(case, seed)
    op, t = case["op"], DTYPE[case["dtype"]]
    if op == "quant":
        v = _exact_quantised(state["x"], case["fmt"])
        return v.clamp(-65504, 65504) if t == torch.float16 else v
    if op == "product":
        y = _exact_packed(state["x"], case["fmt"]) @ _exact_packed(state["w"], case["fmt"]).t()
        return y if state["bias"] is None else y + state["bias"].double()
    x = state["x"].double()
    B, T, C = x.shape
    var, mean = torch.var_mean(x.reshape(B, T, GROUPS, -1), dim=(1, 3), correction=0)
    per = C // GROUPS
    z = (x - mean.repeat_interleave(per, 1)[:, None]) / torch.sqrt(var + EPS).repeat_interleave(per, 1)[:, None]
    z = z * state["gamma"].double() + state["beta"].double()
    if case["silu"]:
        z = z / (1 + torch.exp(-z))
    if op == "norm":
        return z
    y = _exact_quantised(z.to(t).reshape(B * T, C), case["fmt"]) @ _exact_packed(state["w"], case["fmt"]).t()
    return y if state["bias"] is None else y + state["bias"].double()
