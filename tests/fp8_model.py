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


def form(plan, swiglu):
    """What tells the products' code paths apart: CTAs per tile, weight blocks per CTA, accumulators, groups of 128 x scales, scale
    images along K (3: three or more), a tile shared along K, several tiles per CTA."""
    images = -(-plan["kb_split"] // 16)
    return (bool(swiglu), plan["cg"], plan["mt"], plan["nacc"], 1 + (plan["bn"] > 128), min(images, 3), plan["split"] > 1,
            plan["cg"] == 2 and 2 * plan["n_tiles"] * plan["m_tiles"] > plan["grid"])


# A shape for every form that the planner picks for 148 SMs, and a decoder's own.
LINEAR_FORMS = [
    (1, 1, 16), (1, 1, 144), (249, 605, 14448), (518, 1001, 12832), (1298, 1071, 16), (729, 551, 2144), (1097, 611, 4272),
    (3309, 513, 16), (6039, 1311, 1072), (1683, 1303, 2064), (6111, 1297, 2096), (4763, 271, 4432), (1782, 4683, 4224),
    (6271, 513, 16), (6221, 551, 2272), (3627, 1180, 4160), (6323, 527, 16), (3894, 1105, 2080), (6955, 564, 4400),
    (2337, 907, 16), (606, 14789, 1168), (801, 3629, 2080), (845, 9627, 2112), (226, 10155, 4400), (824, 10273, 4528),
    (2856, 1561, 144), (787, 14159, 2016), (4801, 815, 2112), (908, 11665, 2176), (3751, 1027, 4336), (6491, 1809, 4336),
    (1812, 2469, 16), (472, 13039, 2592), (455, 12779, 4752),
    (1, 4096, 4096), (23, 4096, 11008), (512, 4096, 11008), (1537, 5003, 2064), (2048, 4096, 4096), (8192, 11008, 4096)]
SWIGLU_FORMS = [
    (1, 16, 16), (1, 16, 144), (1340, 784, 2080), (295, 16, 14624), (227, 5664, 4144), (993, 400, 8208), (507, 816, 1552),
    (2449, 144, 2064), (1608, 288, 4112), (1833, 912, 16), (1993, 528, 2112), (226, 14448, 2544), (1919, 528, 4160),
    (4961, 832, 4192), (1406, 1232, 16), (258, 4800, 2112), (1576, 1344, 4128), (2717, 3216, 16), (1561, 1520, 2096),
    (1159, 1840, 4176),
    (8, 11008, 4096), (120, 3664, 12880), (300, 2064, 11008), (2048, 11008, 4096)]
