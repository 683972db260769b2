"""The fp8 linears on a B200 against their 64-bit forms: quantiser, norm, product, gate/up product, and a
run of them together, eager, on other streams and captured."""
import ctypes as C
import math

import numpy as np
import pytest
import torch

import fp8_model as F
import ixb_oracle as O
from ignite_xdna_b200 import _lib as L
from ignite_xdna_b200 import fp8

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16, torch.float32]
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}  # half a step, relative


def settle():
    torch.cuda.synchronize()
    L.check(L.load().ixb_device_error(C.byref(C.c_int())))


def randn(*shape, seed, dtype, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (scale * torch.randn(*shape, generator=g, dtype=torch.float64)).to(dtype).cuda()


def same_bits(a, b):
    return torch.equal(a.view(torch.uint8), b.view(torch.uint8))


# ---------------------------------------------------------------- quantise
def check_quantised(x, q, s, rows):
    """x * 2^-e is exact in fp32, so the values and the scales have to be equal."""
    v = x.cpu().double()
    qv, e = F.quantize(v, rows)
    assert torch.equal(F.exponent_of(s.cpu()), e)
    assert torch.equal(torch.nan_to_num(q.cpu().float().double(), nan=1e9), torch.nan_to_num(qv, nan=1e9))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,K", [(1, 16), (1, 128), (3, 144), (17, 4096), (129, 2064), (500, 1040), (2, 16384), (1000, 512)])
@pytest.mark.parametrize("rows", [1, 128])
def test_quantize(M, K, rows, dtype):
    x = randn(M, K, seed=M + K, dtype=dtype, scale=3.0)
    x *= torch.exp2(torch.randint(-9, 9, (M, 1), generator=torch.Generator().manual_seed(1))).to(dtype).cuda()
    q, s = fp8.quantize(x, block_rows=rows)
    settle()
    assert q.dtype is torch.float8_e4m3fn and s.dtype is torch.float8_e8m0fnu
    check_quantised(x, q, s, rows)


@pytest.mark.parametrize("rows", [1, 128])
def test_quantize_borders(rows):
    """Zero blocks, largest values at and next to 448 * 2^k, subnormal inputs, the largest floats,
    infinities and NaN beside ordinary values, and alone in their block."""
    x = torch.zeros(rows * 12, 384, dtype=torch.float32)
    big = [448.0, 449.0, math.nextafter(448.0, 500.0), 448.0 * 2.0 ** -30, 2.0 ** -140, 3.0e38, 1.0, 2.0 ** -126, 1.75 * 2.0 ** -119]
    for i, b in enumerate(big):
        x[i * rows, 5] = b
        x[i * rows, 6] = -b / 3
        x[i * rows, 130] = -b
        x[i * rows, 131] = b / 57
    x[9 * rows, 0] = math.inf
    x[9 * rows, 1] = 2.5
    x[10 * rows, 128] = math.nan
    x[10 * rows, 129] = -17.0
    x[11 * rows, :128] = math.nan
    x[11 * rows, 256] = -math.inf
    x = x.cuda()
    q, s = fp8.quantize(x, block_rows=rows)
    settle()
    check_quantised(x, q, s, rows)


def test_quantize_reads_strided_rows_and_writes_only_its_own():
    wide = randn(40, 640, seed=3, dtype=torch.bfloat16)
    x = wide[:, 64:64 + 272]
    q, s = fp8.quantize(x)
    settle()
    check_quantised(x.contiguous(), q, s, 1)
    lib = L.load()  # the C entry with output strides of its own: what lies between rows stays
    qb = torch.full((40, 304), 0x55, dtype=torch.uint8, device="cuda")
    sb = torch.full((40, 5), 0x55, dtype=torch.uint8, device="cuda")
    L.check(lib.ixb_fp8_quantize(x.data_ptr(), L.BF16, 640, 39, 272, 1, qb.data_ptr(), 304, sb.data_ptr(), 5, None))
    settle()
    assert torch.equal(qb[:39, :272], q.view(torch.uint8)[:39]) and torch.equal(sb[:39, :3], s.view(torch.uint8)[:39])
    assert (qb[:, 272:] == 0x55).all() and (qb[39] == 0x55).all() and (sb[:, 3:] == 0x55).all() and (sb[39] == 0x55).all()


# ---------------------------------------------------------------- norm
# Relative error of y in fp32: the sum of squares has at most 64 serial additions and 10 levels of tree
# (74 roundings, all terms positive) and the product with 1 / K two more, halved by the root; the
# reciprocal root is off by two units in the last place (four roundings), then two products: 44
# roundings of 2^-24 at the most.
Y_ERR = 45 * 2.0 ** -24


def check_normed(x, residual, weight, eps, q, s, h, position):
    h64, y = F.norm(x, residual, weight, eps)
    M, K = x.shape
    if residual is not None:
        assert torch.equal(h, (x.float() + residual.float()).to(x.dtype))
    if position is not None:
        assert s is None and q.dtype is torch.int8
        v = (y * 2.0 ** position).clamp(-128, 127)
        assert ((q.double() - v).abs() <= 0.5 + Y_ERR * v.abs()).all()
        return
    e = F.exponent_of(s)
    top = F.tops(y, 1)
    assert (448 * torch.exp2(e) >= top * (1 - Y_ERR)).all()  # the scale holds the block, and half of it would not
    assert ((448 * torch.exp2(e - 1) < top * (1 + Y_ERR)) | (e == -127)).all()
    scale = torch.exp2(F.spread(e, 1, M, K))
    got = q.float().double() * scale
    assert ((got - y).abs() <= (2.0 ** -4 + 2 * Y_ERR) * y.abs() + 2.0 ** -10 * scale).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,K", [(1, 16), (1, 128), (1, 4096), (5, 144), (31, 5120), (7, 8208), (3, 16384), (2, 32768),
                                 (300, 2064), (400, 4096), (340, 8192), (310, 16400), (2500, 256)])
def test_norm(M, K, dtype):
    x = randn(M, K, seed=M + K, dtype=dtype, scale=2.0)
    r = randn(M, K, seed=M + K + 1, dtype=dtype, scale=5.0)
    w = randn(K, seed=K, dtype=dtype)
    for residual, position in ((r, None), (None, None), (r, 4), (None, 3)):
        q, s, h = fp8.rmsnorm_quant(x, w, eps=1e-5, residual=residual, position=position)
        settle()
        assert (h is None) == (residual is None)
        check_normed(x, residual, w, 1e-5, q, s, h, position)


@pytest.mark.parametrize("M", [3, 500])
def test_norm_with_an_fp32_weight_and_strided_rows(M):
    wide = randn(M, 1024, seed=9, dtype=torch.bfloat16)
    x, r = wide[:, :528], wide[:, 480:480 + 528]
    w = randn(528, seed=2, dtype=torch.float32)
    q, s, h = fp8.rmsnorm_quant(x, w, residual=r)
    settle()
    check_normed(x, r, w, 1e-6, q, s, h, None)


@pytest.mark.parametrize("M", [4, 400])
def test_norm_rows_of_zeros_and_of_what_is_not_finite(M):
    x = randn(M, 512, seed=5, dtype=torch.bfloat16)
    x[0] = 0
    x[1, 7] = math.nan
    x[2, 9] = math.inf
    w = randn(512, seed=6, dtype=torch.bfloat16)
    q, s, _ = fp8.rmsnorm_quant(x, w, eps=0.0 + 1e-6)
    settle()
    assert (q[0].float() == 0).all() and (s[0].view(torch.uint8) == 0).all()
    assert torch.isnan(q[1].float()).all()
    # 1 / sqrt(inf) is 0: the row's finite values are 0 and the infinite one 0 * inf = NaN
    assert torch.isnan(q[2, 9].float()) and (q[2, :9].float() == 0).all() and (q[2, 10:].float() == 0).all()
    check_normed(x[3:], None, w, 1e-6, q[3:], s[3:], None, None)


@pytest.mark.parametrize("M", [1, 700])
def test_norm_in_place(M):
    """h may be the residual or x itself."""
    x = randn(M, 1040, seed=1, dtype=torch.float16)
    r = randn(M, 1040, seed=2, dtype=torch.float16)
    w = randn(1040, seed=3, dtype=torch.float16)
    q0, s0, h0 = fp8.rmsnorm_quant(x, w, residual=r)
    for at in (x.clone(), r.clone()):
        own_x, own_r = (at, r) if torch.equal(at, x) else (x, at)
        q, s = torch.empty_like(q0), torch.empty((M, 9), dtype=s0.dtype, device="cuda")
        L.check(L.load().ixb_rmsnorm_quant(own_x.data_ptr(), 1040, own_r.data_ptr(), 1040, w.data_ptr(), L.F16, L.F16, M, 1040, 1e-6,
                                           0, at.data_ptr(), 1040, q.data_ptr(), 1040, s.data_ptr(), 9, None))
        settle()
        assert torch.equal(at, h0) and same_bits(q, q0) and same_bits(s, s0)


@pytest.mark.parametrize("M,K", [(1, 144), (3, 2064), (400, 272), (310, 16400)])
def test_norm_writes_only_its_own(M, K):
    x = randn(M, K, seed=1, dtype=torch.bfloat16)
    r = randn(M, K, seed=2, dtype=torch.bfloat16)
    w = randn(K, seed=3, dtype=torch.bfloat16)
    q, s, h = fp8.rmsnorm_quant(x, w, residual=r)
    nb = -(-K // 128)
    qb = torch.full((M + 1, K + 48), 0x55, dtype=torch.uint8, device="cuda")
    sb = torch.full((M + 1, nb + 2), 0x55, dtype=torch.uint8, device="cuda")
    hb = torch.full((M + 1, K + 24), 7.0, dtype=torch.bfloat16, device="cuda")
    L.check(L.load().ixb_rmsnorm_quant(x.data_ptr(), K, r.data_ptr(), K, w.data_ptr(), L.BF16, L.BF16, M, K, 1e-6, 0, hb.data_ptr(),
                                       K + 24, qb.data_ptr(), K + 48, sb.data_ptr(), nb + 2, None))
    settle()
    assert torch.equal(qb[:M, :K], q.view(torch.uint8)) and torch.equal(sb[:M, :nb], s.view(torch.uint8)) and torch.equal(hb[:M, :K], h)
    assert (qb[:, K:] == 0x55).all() and (qb[M] == 0x55).all() and (sb[:, nb:] == 0x55).all() and (sb[M] == 0x55).all()
    assert (hb[:, K:] == 7).all() and (hb[M] == 7).all()


# ---------------------------------------------------------------- product
def slack(K, total):
    """Error of an fp32 sum of K exact products whose absolute values add up to `total`, each addition
    off by at most 2^-23 of a partial sum (a tensor core may cut instead of rounding)."""
    return K * 2.0 ** -23 * total


def check_product(x, xs, w, ws, out):
    ref, total = F.product(x, xs, w, ws)
    err = (out.double() - ref).abs()
    assert (err <= HALF[out.dtype] * ref.abs() + slack(x.shape[1], total)).all()
    # All together: each of K additions is off by at most 2^-23 of the running sum, and a cutting adder errs one
    # way. After k of K terms of random signs the running sums' norm is sqrt(k / K) of the whole, and
    # sum over k of sqrt(k / K) is at most (2 / 3) K + 1.
    K = x.shape[1]
    assert err.norm() <= (HALF[out.dtype] + 2.0 ** -23 * (K / 1.5 + 1)) * ref.norm()


SHAPES = [(1, 1, 16), (1, 16, 128), (1, 128, 144), (1, 4096, 4096), (1, 5003, 528), (2, 256, 11008), (7, 640, 1040),
          (16, 512, 512), (17, 1000, 2064), (23, 4096, 1024), (33, 300, 4096), (64, 2048, 2048), (100, 384, 128),
          (127, 513, 640), (128, 4096, 512), (200, 1024, 8192), (255, 130, 272), (257, 2049, 1040), (512, 4096, 1024),
          (1000, 520, 400), (1537, 2501, 912), (2048, 1024, 1536), (4096, 128, 256), (300, 16, 65536), (3000, 6000, 512)]


@pytest.mark.parametrize("M,N,K", SHAPES)
def test_linear(M, N, K):
    x, xs = F.make(M, K, 1, seed=M + K, device="cuda")
    w, ws = F.make(N, K, 128, seed=N + K, device="cuda")
    for dtype in TYPES:
        out = fp8.linear(x, xs, w, ws, out_dtype=dtype)
        settle()
        assert out.shape == (M, N) and out.dtype is dtype
        check_product(x, xs, w, ws, out)


@pytest.mark.parametrize("M", [3, 90, 700])
def test_linear_with_strided_operands(M):
    """x, w and out as parts of wider matrices, scales with odd strides and addresses."""
    K, N = 528, 391
    x, xs = F.make(M, K, 1, seed=1, device="cuda")
    w, ws = F.make(N, K, 128, seed=2, device="cuda")
    ref = fp8.linear(x, xs, w, ws)
    wide_x = torch.zeros(M, 1024, dtype=torch.uint8, device="cuda")
    wide_x[:, 48:48 + K] = x.view(torch.uint8)
    wide_w = torch.full((N, 640), 0x7F, dtype=torch.uint8, device="cuda")
    wide_w[:, 16:16 + K] = w.view(torch.uint8)
    wide_xs = torch.full((M, 7), 255, dtype=torch.uint8, device="cuda")
    wide_xs[:, 1:6] = xs.view(torch.uint8)
    wide_ws = torch.full((4, 11), 255, dtype=torch.uint8, device="cuda")
    wide_ws[:, 3:8] = ws.view(torch.uint8)
    out = torch.full((M + 1, N + 5), 7.0, dtype=torch.bfloat16, device="cuda")
    fp8.linear(wide_x.view(fp8.E4M3)[:, 48:48 + K], wide_xs.view(fp8.E8M0)[:, 1:6], wide_w.view(fp8.E4M3)[:, 16:16 + K],
               wide_ws.view(fp8.E8M0)[:, 3:8], out=out[:M, 3:3 + N])
    settle()
    assert torch.equal(out[:M, 3:3 + N], ref)
    assert (out[:, :3] == 7).all() and (out[:, 3 + N:] == 7).all() and (out[M] == 7).all()


@pytest.mark.parametrize("M", [5, 600])
def test_linear_nan_stays_in_its_row_and_block(M):
    K, N = 400, 300
    x, xs = F.make(M, K, 1, seed=11, device="cuda")
    w, ws = F.make(N, K, 128, seed=12, device="cuda")
    ref = fp8.linear(x, xs, w, ws)
    x.view(torch.uint8)[1, 37] = 0x7F          # NaN value: row 1
    xs.view(torch.uint8)[3, 2] = 255           # NaN scale: row 3
    ws.view(torch.uint8)[1, 0] = 255           # NaN scale of weight rows 128 .. 255
    out = fp8.linear(x, xs, w, ws)
    settle()
    nan = torch.zeros(M, N, dtype=torch.bool, device="cuda")
    nan[1], nan[3], nan[:, 128:256] = True, True, True
    assert torch.equal(torch.isnan(out), nan)
    assert torch.equal(out[~nan], ref[~nan])


@pytest.mark.parametrize("M", [2, 300])
def test_linear_scale_range(M):
    """Scales from 2^-100 to 2^100 on both sides: the products' exponents add up, large times small."""
    K, N = 1024, 256
    x, xs = F.make(M, K, 1, seed=21, device="cuda", spread_log2=0.0)
    w, ws = F.make(N, K, 128, seed=22, device="cuda", spread_log2=0.0)
    e = torch.randint(-100, 101, (1, K // 128), generator=torch.Generator().manual_seed(3)).cuda()
    xs = (e + 127).to(torch.uint8).expand(M, -1).contiguous().view(fp8.E8M0)
    ws = (-e + 127).to(torch.uint8).expand(2, -1).contiguous().view(fp8.E8M0)
    out = fp8.linear(x, xs, w, ws, out_dtype=torch.float32)
    settle()
    check_product(x, xs, w, ws, out)


def test_linear_largest_values():
    """+-448 everywhere: the largest sums."""
    for M in (1, 130):
        x = torch.full((M, 4096), 448.0, device="cuda").to(fp8.E4M3)
        w = torch.full((256, 4096), -448.0, device="cuda").to(fp8.E4M3)
        xs = torch.full((M, 32), 127, dtype=torch.uint8, device="cuda").view(fp8.E8M0)
        ws = torch.full((2, 32), 127, dtype=torch.uint8, device="cuda").view(fp8.E8M0)
        out = fp8.linear(x, xs, w, ws, out_dtype=torch.float32)
        settle()
        assert (out == -448.0 * 448.0 * 4096).all()


@pytest.mark.parametrize("sms", ["4", "16"])
def test_products_with_many_tiles_per_cta(sms, monkeypatch):
    """A planner SM count below the tile count: each CTA runs several tiles, with one accumulator and with two."""
    monkeypatch.setenv("IXB_SM_COUNT", sms)
    for M, N, K in [(1000, 700, 656), (40, 4096, 256), (2000, 1024, 1280)]:
        x, xs = F.make(M, K, 1, seed=M, device="cuda")
        w, ws = F.make(N, K, 128, seed=N, device="cuda")
        out = fp8.linear(x, xs, w, ws)
        settle()
        check_product(x, xs, w, ws, out)
        if N % 16 == 0:
            u, us = F.make(N, K, 128, seed=N + 1, device="cuda")
            q, s = fp8.linear_swiglu(x, xs, w, ws, u, us)
            settle()
            check_swiglu(x, xs, w, ws, u, us, q, s)


# ---------------------------------------------------------------- gate and up
def check_swiglu(x, xs, g, gs, u, us, q, s):
    gate, gt = F.product(x, xs, g, gs)
    up, ut = F.product(x, xs, u, us)
    M, N = gate.shape
    y = gate * torch.sigmoid(gate) * up
    # the products' errors through silu (its slope is below 1.1) and the product, and the few roundings of
    # the exponential (relative 2^-22 and 2^-24 of its argument), the quotient and the products
    K = x.shape[1]
    err = 1.1 * slack(K, gt) * (up.abs() + slack(K, ut)) + (gate * torch.sigmoid(gate)).abs() * slack(K, ut)
    err = err + y.abs() * (2.0 ** -20 + 2.0 ** -22 * gate.abs().clamp(max=90))
    e = F.exponent_of(s)
    top, off = F.tops(y, 1), F.tops(err, 1)
    assert (448 * torch.exp2(e) >= top - off).all()
    assert ((448 * torch.exp2(e - 1) < top + off) | (e == -127)).all()
    scale = torch.exp2(F.spread(e, 1, M, N))
    got = q.float().double() * scale
    assert ((got - y).abs() <= 2.0 ** -4 * (y.abs() + err) + err + 2.0 ** -10 * scale).all()


@pytest.mark.parametrize("M,N,K", [(1, 16, 16), (1, 11008, 512), (2, 144, 4096), (8, 1024, 4096), (17, 528, 272), (50, 128, 128),
                                   (64, 2048, 1024), (120, 272, 4096), (129, 400, 912), (500, 1040, 640), (1111, 2064, 528),
                                   (2048, 5504, 256), (4000, 128, 1024)])
def test_linear_swiglu(M, N, K):
    x, xs = F.make(M, K, 1, seed=M + K, device="cuda")
    g, gs = F.make(N, K, 128, seed=N + K, device="cuda")
    u, us = F.make(N, K, 128, seed=N + K + 1, device="cuda")
    # gates of a few units, where the sigmoid is neither 0 nor 1
    gs = (gs.view(torch.uint8) - int(round(math.log2(math.sqrt(K))))).view(fp8.E8M0)
    us = (us.view(torch.uint8) - int(round(math.log2(math.sqrt(K))))).view(fp8.E8M0)
    q, s = fp8.linear_swiglu(x, xs, g, gs, u, us)
    settle()
    check_swiglu(x, xs, g, gs, u, us, q, s)


def test_linear_swiglu_large_gates_and_nan():
    """Gates of +-1000s (the exponential overflows to infinity and underflows to 0), and a NaN row."""
    for M in (6, 300):
        K, N = 256, 256
        x, xs = F.make(M, K, 1, seed=1, device="cuda")
        g, gs = F.make(N, K, 128, seed=2, device="cuda")
        u, us = F.make(N, K, 128, seed=3, device="cuda")
        gs = (gs.view(torch.uint8) + 7).view(fp8.E8M0)
        x.view(torch.uint8)[2, 3] = 0x7F
        q, s = fp8.linear_swiglu(x, xs, g, gs, u, us)
        settle()
        assert torch.isnan(q[2].float()).all() and (s[2].view(torch.uint8) == 0).all()
        keep = torch.arange(M, device="cuda") != 2
        assert torch.isfinite(q[keep].float()).all()
        check_swiglu(x[keep], xs[keep], g, gs, u, us, q[keep], s[keep])


@pytest.mark.parametrize("M,N", [(1, 144), (5, 2064), (33, 272), (130, 144), (300, 2064), (700, 272)])
def test_linear_swiglu_writes_only_its_own(M, N):
    """Padded outputs with a guard row: what lies between and behind the rows stays as it was, in both forms
    and with a last block of 16 outputs."""
    K = 272
    x, xs = F.make(M, K, 1, seed=1, device="cuda")
    g, gs = F.make(N, K, 128, seed=2, device="cuda")
    u, us = F.make(N, K, 128, seed=3, device="cuda")
    q, s = fp8.linear_swiglu(x, xs, g, gs, u, us)
    nb = -(-N // 128)
    qb = torch.full((M + 1, N + 32), 0x55, dtype=torch.uint8, device="cuda")
    sb = torch.full((M + 1, nb + 3), 0x55, dtype=torch.uint8, device="cuda")
    L.check(L.load().ixb_fp8_linear_swiglu(x.data_ptr(), K, xs.data_ptr(), xs.stride(0), g.data_ptr(), K, gs.data_ptr(), gs.stride(0),
                                           u.data_ptr(), K, us.data_ptr(), us.stride(0), qb.data_ptr(), N + 32, sb.data_ptr(), nb + 3,
                                           M, N, K, None))
    settle()
    assert torch.equal(qb[:M, :N], q.view(torch.uint8)) and torch.equal(sb[:M, :nb], s.view(torch.uint8))
    assert (qb[:, N:] == 0x55).all() and (qb[M] == 0x55).all() and (sb[:, nb:] == 0x55).all() and (sb[M] == 0x55).all()


@pytest.mark.parametrize("M", [1, 40, 500])
def test_gate_and_up_as_views_of_one_weight(M):
    K, N = 528, 400
    x, xs = F.make(M, K, 1, seed=1, device="cuda")
    g, gs = F.make(N, K, 128, seed=2, device="cuda")
    u, us = F.make(N, K, 128, seed=3, device="cuda")
    both = torch.cat([g.view(torch.uint8), u.view(torch.uint8)]).view(fp8.E4M3)
    q, s = fp8.linear_swiglu(x, xs, both[:N], gs, both[N:], us)
    q1, s1 = fp8.linear_swiglu(x, xs, g, gs, u, us)
    settle()
    assert same_bits(q, q1) and same_bits(s, s1)


# ---------------------------------------------------------------- together
def layer(tokens, hidden, inner, seed):
    """Weights and inputs of norm -> gate/up -> down."""
    weights = [fp8.quantize(randn(n, k, seed=seed + i, dtype=torch.bfloat16, scale=k ** -0.5), block_rows=128)
               for i, (n, k) in enumerate([(inner, hidden), (inner, hidden), (hidden, inner)])]
    x = randn(tokens, hidden, seed=seed + 5, dtype=torch.bfloat16)
    r = randn(tokens, hidden, seed=seed + 6, dtype=torch.bfloat16, scale=3.0)
    return weights, x, r, randn(hidden, seed=seed + 7, dtype=torch.bfloat16)


def mlp(weights, x, r, nw):
    (g, gs), (u, us), (d, ds) = weights
    q, s, h = fp8.rmsnorm_quant(x, nw, residual=r)
    q2, s2 = fp8.linear_swiglu(q, s, g, gs, u, us)
    return fp8.linear(q2, s2, d, ds), h, (q, s, q2, s2)


@pytest.mark.parametrize("tokens", [1, 20, 333])
def test_a_decoder_mlp(tokens):
    """Norm, gate/up and down as a decoder layer calls them: each step against its 64-bit form on what the step
    before it gave, and the same bits every time."""
    weights, x, r, nw = layer(tokens, 1024, 2816, seed=tokens)
    (g, gs), (u, us), (d, ds) = weights
    out, h, (q, s, q2, s2) = mlp(weights, x, r, nw)
    settle()
    check_normed(x, r, nw, 1e-6, q, s, h, None)
    check_swiglu(q, s, g, gs, u, us, q2, s2)
    check_product(q2, s2, d, ds, out)
    for _ in range(3):  # no sum depends on the order in which CTAs finish
        again, _, (a, b, c, e) = mlp(weights, x, r, nw)
        assert torch.equal(again, out) and all(same_bits(i, j) for i, j in ((a, q), (b, s), (c, q2), (e, s2)))


@pytest.mark.parametrize("tokens", [1, 200])
def test_a_decoder_mlp_on_other_streams_and_in_a_graph(tokens):
    weights, x, r, nw = layer(tokens, 512, 1408, seed=40 + tokens)
    ref = mlp(weights, x, r, nw)[0]
    torch.cuda.synchronize()
    side = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for _ in range(4):  # two calls at once, on two streams
        for st in side:
            with torch.cuda.stream(st):
                outs.append(mlp(weights, x, r, nw)[0])
    torch.cuda.synchronize()
    assert all(torch.equal(o, ref) for o in outs)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = mlp(weights, x, r, nw)[0]
    x2 = randn(tokens, 512, seed=99, dtype=torch.bfloat16)
    want = mlp(weights, x2, r, nw)[0]
    x.copy_(x2)
    for _ in range(3):
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
    settle()


def test_the_first_calls_of_a_process_may_be_captured():
    """Nothing that a first call sets up (kernel attributes, the tensor-map encoder) is closed to a capture."""
    code = """
import torch
from ignite_xdna_b200 import fp8
x = torch.randn(5, 512, device="cuda").bfloat16()
many = torch.randn(400, 512, device="cuda").bfloat16()
w = torch.randn(256, 512, device="cuda").bfloat16()
nw = torch.ones(512, device="cuda").bfloat16()
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
def step(x):
    wq, ws = fp8.quantize(w, block_rows=128)
    q, s, _ = fp8.rmsnorm_quant(x, nw)
    q2, s2 = fp8.linear_swiglu(q, s, wq, ws, wq, ws)
    return fp8.linear(q, s, wq, ws), q2, s2
with torch.cuda.graph(g):
    outs = step(x) + step(many)
g.replay()
torch.cuda.synchronize()
for a, b in zip(outs, step(x) + step(many)):
    assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
print("captured")
"""
    import subprocess
    import sys
    from pathlib import Path
    r = subprocess.run([sys.executable, "-c", code], cwd=Path(__file__).resolve().parent.parent, capture_output=True, text=True,
                       timeout=300)
    assert r.returncode == 0 and "captured" in r.stdout, r.stderr


def test_the_int8_norm_feeds_the_w4a8_product():
    M, K, N = 37, 1024, 272
    x = randn(M, K, seed=1, dtype=torch.bfloat16)
    w = randn(K, seed=2, dtype=torch.bfloat16)
    q, _, _ = fp8.rmsnorm_quant(x, w, position=5)
    rng = np.random.default_rng(4)
    w4 = O.pack_int4(rng.integers(-8, 8, size=(K, N), dtype=np.int8))
    gpos = (5 + rng.integers(0, 4, size=(K // 128, N))).astype(np.int8)
    shift = rng.integers(6, 14, size=N).astype(np.int32)
    lib = L.load()
    nbytes = C.c_uint64()
    L.check(lib.ixb_w4a8_image_bytes(K, N, C.byref(nbytes)))
    img = torch.empty(nbytes.value, dtype=torch.uint8, device="cuda")
    dw, dg, ds = (torch.from_numpy(a).cuda() for a in (w4, gpos, shift))
    L.check(lib.ixb_w4a8_prepare(dw.data_ptr(), dg.data_ptr(), K, N, img.data_ptr(), None))
    out = torch.empty((M, N), dtype=torch.int8, device="cuda")
    L.check(lib.ixb_w4a8_gemm(q.data_ptr(), img.data_ptr(), ds.data_ptr(), out.data_ptr(), M, N, K, None))
    settle()
    assert np.array_equal(out.cpu().numpy(), O.w4a8_srs(q.cpu().numpy(), w4, gpos, shift))


# ---------------------------------------------------------------- calls
def test_no_rows():
    w, ws = F.make(256, 512, 128, 1, device="cuda")
    x = torch.empty(0, 512, dtype=torch.bfloat16, device="cuda")
    q, s, h = fp8.rmsnorm_quant(x, torch.ones(512, dtype=torch.bfloat16, device="cuda"), residual=x)
    assert q.shape == (0, 512) and s.shape == (0, 4) and h.shape == (0, 512)
    q, s = fp8.quantize(x)
    assert fp8.linear(q, s, w, ws).shape == (0, 256)
    q, s = fp8.linear_swiglu(q, s, w, ws, w, ws)
    assert q.shape == (0, 256) and s.shape == (0, 2)
    settle()


def test_refusals():
    x, xs = F.make(4, 512, 1, 0, device="cuda")
    w, ws = F.make(256, 512, 128, 1, device="cuda")
    b = torch.zeros(4, 512, dtype=torch.bfloat16, device="cuda")
    nw = torch.ones(512, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(TypeError):
        fp8.linear(b, xs, w, ws)
    with pytest.raises(TypeError):
        fp8.linear(x, xs.view(torch.uint8), w, ws)
    with pytest.raises(ValueError):
        fp8.linear(x, xs[:, :3], w, ws)
    with pytest.raises(ValueError):
        fp8.linear(x, xs, w[:, :256], ws)
    with pytest.raises(ValueError):
        fp8.linear(x, xs, w, ws[:1])
    with pytest.raises(ValueError):
        fp8.linear(x[0], xs, w, ws)
    with pytest.raises(ValueError):
        fp8.linear(x, xs, w, ws.cpu())
    with pytest.raises(ValueError):
        fp8.linear(x.t().contiguous().t(), xs, w, ws)
    with pytest.raises(TypeError):
        fp8.linear(x, xs, w, ws, out_dtype=torch.float64)
    with pytest.raises(ValueError):
        fp8.linear(x, xs, w, ws, out=torch.empty(4, 255, dtype=torch.bfloat16, device="cuda"))
    with pytest.raises(L.IxbError):  # rows that start off the 16-byte grid
        fp8.linear(torch.empty(4, 1024, dtype=torch.uint8, device="cuda").view(fp8.E4M3)[:, 8:520], xs, w, ws)
    with pytest.raises(ValueError):
        fp8.linear_swiglu(x, xs, w, ws, w[:128], ws[:1])
    with pytest.raises(L.IxbError):
        fp8.linear_swiglu(x, xs, w[:200], ws, w[:200], ws)
    with pytest.raises(L.IxbError):
        fp8.quantize(b, block_rows=2)
    with pytest.raises(L.IxbError):
        fp8.quantize(b[:, :100])
    with pytest.raises(TypeError):
        fp8.rmsnorm_quant(b, nw.half())
    with pytest.raises(ValueError):
        fp8.rmsnorm_quant(b, nw[:256])
    with pytest.raises(TypeError):
        fp8.rmsnorm_quant(b, nw, residual=b.float())
    with pytest.raises(ValueError):
        fp8.rmsnorm_quant(b, nw, residual=b[:2])
    with pytest.raises(L.IxbError):
        fp8.rmsnorm_quant(b, nw, eps=-1.0)
    with pytest.raises(L.IxbError):
        fp8.rmsnorm_quant(b, nw, position=99)
    settle()


def test_two_devices_in_one_process():
    if torch.cuda.device_count() < 2:
        pytest.skip("one GPU is visible")
    for dev in ("cuda:0", "cuda:1"):  # the current device stays 0
        x, xs = F.make(40, 512, 1, 0, device=dev)
        w, ws = F.make(256, 512, 128, 1, device=dev)
        out = fp8.linear(x, xs, w, ws)
        torch.cuda.synchronize(dev)
        assert out.device == x.device
        check_product(x, xs, w, ws, out)
    with pytest.raises(ValueError, match="cuda"):
        fp8.linear(x, xs, w.to("cuda:0"), ws)


def test_what_requires_grad_is_refused_and_no_grad_allows_it():
    x = randn(3, 256, seed=1, dtype=torch.bfloat16)
    w = torch.nn.Parameter(torch.ones(256, dtype=torch.bfloat16, device="cuda"))
    with pytest.raises(ValueError, match="grad"):
        fp8.rmsnorm_quant(x, w)
    with torch.no_grad():
        q, s, _ = fp8.rmsnorm_quant(x, w)
    settle()
    assert not q.requires_grad


def test_an_inference_mode_tensor_and_a_single_row_view():
    """Rows of one, whose stride says nothing, and tensors without autograd state."""
    with torch.inference_mode():
        x, xs = F.make(5, 512, 1, 0, device="cuda")
        w, ws = F.make(256, 512, 128, 1, device="cuda")
        every = fp8.linear(x, xs, w, ws)
        one = fp8.linear(x[2:3], xs[2:3], w, ws)
        settle()
        assert torch.equal(one, every[2:3])


def test_out_that_shares_memory_with_an_input_is_refused():
    x, xs = F.make(64, 512, 1, 0, device="cuda")
    w, ws = F.make(256, 512, 128, 1, device="cuda")
    buf = torch.zeros(256 * 512, dtype=torch.uint8, device="cuda")
    out = buf.view(torch.bfloat16)[-64 * 256:].view(64, 256)
    shared = buf.view(torch.float8_e4m3fn).view(256, 512)
    shared.copy_(w)
    before = buf.clone()
    with pytest.raises(ValueError, match="shares memory"):
        fp8.linear(x, xs, shared, ws, out=out)
    settle()
    assert torch.equal(buf, before)
    head = buf.view(torch.float8_e4m3fn)[:128 * 512].view(128, 512)  # beside it in one buffer is no overlap
    tail = buf.view(torch.bfloat16)[-64 * 128:].view(64, 128)
    fp8.linear(x, xs, head, ws[:1], out=tail)
    settle()
    assert torch.equal(tail, fp8.linear(x, xs, w[:128], ws[:1]))


def test_writing_out_is_seen_by_autograd():
    """A tensor that a graph has saved is written: the backward pass raises and does not use the new values."""
    x, xs = F.make(8, 256, 1, 0, device="cuda")
    w, ws = F.make(128, 256, 128, 1, device="cuda")
    out = torch.ones(8, 128, dtype=torch.float32, device="cuda")
    leaf = torch.ones(8, 128, device="cuda", requires_grad=True)
    y = (leaf * out).sum()
    fp8.linear(x, xs, w, ws, out=out)
    settle()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
    with torch.inference_mode():  # tensors without a version
        fp8.linear(x, xs, w, ws, out=torch.empty(8, 128, device="cuda"))
    settle()
