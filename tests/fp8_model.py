"""64-bit forms of the fp8 operators, from their definitions, for the tests."""
import math

import torch

BLOCK = 128
F64 = torch.float64


def e4m3(v):
    """Nearest e4m3 value of float64 v, ties to even: 3 fraction bits, steps of 2**-9 below 2**-6."""
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(v / step) * step


def tops(v, rows):
    """The largest finite |v| of each block [ceil(M / rows), ceil(K / 128)]."""
    M, K = v.shape
    mb, kb = -(-M // rows), -(-K // BLOCK)
    wide = torch.zeros(mb * rows, kb * BLOCK, dtype=F64, device=v.device)
    wide[:M, :K] = torch.where(torch.isfinite(v), v.abs(), 0.0)
    return wide.view(mb, rows, kb, BLOCK).amax(dim=(1, 3))


def exponents(top):
    """The least e >= -127 with 448 * 2**e >= top."""
    e = torch.full_like(top, -127.0)
    for k in range(-126, 125):
        e = torch.where(top > 448.0 * 2.0 ** (k - 1), float(k), e)
    return e


def spread(s, rows, M, K):
    """Per-block values as [M, K]."""
    return s.repeat_interleave(rows, 0)[:M].repeat_interleave(BLOCK, 1)[:, :K]


def quantize(v, rows):
    """(values of q, exponents) of float64 v; what is not finite is NaN."""
    M, K = v.shape
    e = exponents(tops(v, rows))
    q = e4m3(torch.where(torch.isfinite(v), v, 0.0) * torch.exp2(-spread(e, rows, M, K)))
    return torch.where(torch.isfinite(v), q, math.nan), e


def exponent_of(scale):
    return scale.view(torch.uint8).double() - 127


def values(q, scale, rows):
    return q.float().double() * torch.exp2(spread(exponent_of(scale), rows, *q.shape))


def norm(x, residual, weight, eps):
    h = x.double() + (0 if residual is None else residual.double())
    return h, h / torch.sqrt((h * h).mean(1, keepdim=True) + eps) * weight.double()


def product(x, xs, w, ws):
    """(x . w^T, sum of the terms' absolute values)."""
    a, b = values(x, xs, 1), values(w, ws, BLOCK)
    return a @ b.t(), a.abs() @ b.abs().t()


def make(M, K, rows, seed, device="cpu", spread_log2=4.0):
    """An e4m3 matrix with scales as a quantiser gives them: normal values, blocks of different sizes."""
    g = torch.Generator().manual_seed(seed)
    v = torch.randn(M, K, generator=g, dtype=F64)
    size = torch.exp2(spread_log2 * (torch.rand(-(-M // rows), -(-K // BLOCK), generator=g, dtype=F64) - 0.5))
    q, e = quantize(v * spread(size, rows, M, K), rows)
    return (q.float().to(torch.float8_e4m3fn).to(device),
            (e + 127).to(torch.uint8).view(torch.float8_e8m0fnu).to(device))
