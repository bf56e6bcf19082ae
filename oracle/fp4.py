"""CPU restatement of the 4-bit floating-point formats in 64 bits (for the tests only; the package never imports it).

mx: one E8M0 scale per 32 elements, 2^(floor(log2 max) - 2).  nv: one E4M3 scale per 16 elements, e4m3(max / (6 s_row)), under
a power of two per row, the smallest with row max <= 2688 s_row.  Codes are E2M1, nearest, ties to even.
"""
import torch

E2M1 = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64)
E4M3 = torch.tensor([(k * 2.0 ** -9) if k < 8 else (1 + (k % 8) / 8) * 2.0 ** (k // 8 - 7) for k in range(127)], dtype=torch.float64)
BLOCK = {"mx": 32, "nv": 16}


def nearest(v, grid):
    """Index of the nearest grid value, a tie going to the even index; beyond the end the last."""
    hi = torch.searchsorted(grid, v.contiguous()).clamp(max=len(grid) - 1)
    lo = (hi - 1).clamp(min=0)
    below, above = v - grid[lo], grid[hi] - v
    return torch.where((below < above) | ((below == above) & (lo % 2 == 0)), lo, hi)


def quantise(x, fmt):
    """(codes 0 .. 15 as int64 [M,K], scale bytes int64 [M, K / block], row scales fp64 [M] or None) of finite rows."""
    M, K = x.shape
    b = x.double().reshape(M, -1, BLOCK[fmt])
    amax = b.abs().amax(dim=2)
    row = None
    if fmt == "mx":
        e = torch.frexp(amax)[1].long() - 3                       # floor(log2) - 2
        byte = torch.where(amax > 0, e + 127, torch.zeros_like(e)).clamp(min=0)
        s = torch.ldexp(torch.ones_like(amax), byte - 127)
    else:
        m, e = torch.frexp(amax.amax(dim=1) / 2688)
        e = torch.where(m == 0.5, e - 1, e)
        e = torch.where(amax.amax(dim=1) > 0, e.clamp(min=-100), torch.zeros_like(e))
        row = torch.ldexp(torch.ones_like(m), e)
        byte = nearest(amax / row[:, None] / 6, E4M3)
        s = E4M3[byte] * row[:, None]
    s = s[:, :, None]
    q = torch.where(s > 0, b.abs() / torch.where(s > 0, s, torch.ones_like(s)), torch.zeros_like(b))
    code = nearest(q, E2M1)
    code = torch.where(torch.signbit(b) & (s > 0), code + 8, code)
    return code.reshape(M, K), byte, row


def pack(code):
    c = code.to(torch.uint8)
    return c[:, 0::2] | (c[:, 1::2] << 4)


def unpack(codes):
    return torch.stack([codes & 15, codes >> 4], dim=2).reshape(codes.shape[0], -1).long()


def untile(scales, M, K, fmt):
    """Scale bytes [M, K / block] out of the tiled array, byte by byte."""
    blk = torch.arange(K // BLOCK[fmt])[None, :]
    r = torch.arange(M)[:, None]
    return scales[r // 128, blk // 4, (r % 32) * 16 + (r // 32 % 4) * 4 + blk % 4].long()


def values(code, byte, row, fmt):
    """64-bit values; the E8M0 NaN (255) and a NaN row scale give NaN."""
    v = torch.where(code >= 8, -E2M1[code % 8], E2M1[code % 8]).reshape(code.shape[0], -1, BLOCK[fmt])
    if fmt == "mx":
        s = torch.ldexp(torch.ones_like(byte, dtype=torch.float64), byte - 127)
        s = torch.where(byte == 255, torch.full_like(s, float("nan")), s)
    else:
        s = E4M3[byte] * row.double()[:, None]
    return (v * s[:, :, None]).reshape(code.shape)


def packed_values(codes, scales, row, fmt):
    """64-bit values of packed rows as the library keeps them (CPU tensors)."""
    M, K = codes.shape[0], codes.shape[1] * 2
    return values(unpack(codes), untile(scales, M, K, fmt), row, fmt)
