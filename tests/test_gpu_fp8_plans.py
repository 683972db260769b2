"""The fp8 products in every form that the planner picks, at a decoder's depths: chains of launches, scale images
that follow one another, accuracy of the 32-bit sums."""
import math

import pytest
import torch

import fp8_model as F
from ignite_xdna_b200 import fp8
from test_fp8 import plan
from test_gpu_fp8 import check_product, check_swiglu, layer, mlp, same_bits, settle

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------- launches one after another
def test_launches_that_take_over_one_anothers_sms():
    """Pairs with one tile and with several, between few-token products, norms and quantisers, enqueued without a wait: each launch
    gets shared memory and TMEM that the one before has just left, and has to find its own barriers as it set them."""
    K, N = 2064, 1040
    w, ws = F.make(N, K, 128, 1, device="cuda")
    u, us = F.make(N, K, 128, 2, device="cuda")
    nw = torch.ones(K, dtype=torch.bfloat16, device="cuda")
    sets = []
    for tokens in (1, 40, 300, 1000, 3000):
        x, xs = F.make(tokens, K, 1, tokens, device="cuda")
        sets.append((x, xs, torch.randn(tokens, K, device="cuda").bfloat16()))

    def calls(x, xs, b):
        q, s, _ = fp8.rmsnorm_quant(b, nw)
        return [fp8.linear(x, xs, w, ws), *fp8.linear_swiglu(x, xs, w, ws, u, us), fp8.linear(q, s, w, ws), *fp8.quantize(b)]

    want = []
    for one in sets:
        want.append(calls(*one))
        settle()
    for turn in range(40):
        order = sets[turn % 5:] + sets[:turn % 5]
        got = [calls(*one) for one in order]
        settle()
        for g, e in zip(got, want[turn % 5:] + want[:turn % 5]):
            assert all(same_bits(a, b) for a, b in zip(g, e))


# ---------------------------------------------------------------- out=
def test_padded_out_over_an_input_is_refused_and_beside_it_is_not():
    """Views of wider matrices: refused where a byte is shared with an operand or its scales, taken where the columns
    of one matrix are divided between them."""
    M, N, K = 40, 64, 512
    x, xs = F.make(M, K, 1, 0, device="cuda")
    w, ws = F.make(N, K, 128, 1, device="cuda")
    want = fp8.linear(x, xs, w, ws)
    buf = torch.zeros(64, 1024, dtype=torch.uint8, device="cuda")
    buf[:M, :K] = x.view(torch.uint8)
    wide_x = buf[:M, :K].view(fp8.E4M3)
    before = buf.clone()
    bf16 = buf.view(torch.bfloat16)
    for rows, out in ((slice(0, M), bf16[:M, 224:288]), (slice(0, M), bf16[:M, 0:64]), (slice(0, 24), bf16[23:47, 255:319])):
        with pytest.raises(ValueError, match="shares memory"):
            fp8.linear(wide_x[rows], xs[rows], w, ws, out=out)
    buf_w = torch.zeros(N, 1024, dtype=torch.uint8, device="cuda")
    buf_w[:, 512:] = w.view(torch.uint8)
    with pytest.raises(ValueError, match="shares memory"):
        fp8.linear(x, xs, buf_w[:, 512:].view(fp8.E4M3), ws, out=buf_w.view(torch.bfloat16)[:M, 200:264])
    buf_s = torch.zeros(M, 132, dtype=torch.uint8, device="cuda")
    buf_s[:, 126:130] = xs.view(torch.uint8)
    with pytest.raises(ValueError, match="shares memory"):
        fp8.linear(x, buf_s[:, 126:130].view(fp8.E8M0), w, ws, out=buf_s.view(torch.bfloat16)[:, :64])
    settle()
    assert torch.equal(buf, before)
    out = bf16[:M, 256:320]  # beside x in the same rows
    assert fp8.linear(wide_x, xs, w, ws, out=out).data_ptr() == out.data_ptr()
    settle()
    assert torch.equal(out, want) and torch.equal(buf[:M, :K], before[:M, :K])


# ---------------------------------------------------------------- every form, at a decoder's depths
def make(M, K, rows, seed):
    """As fp8_model.make, on the GPU: normal values, blocks of different sizes."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    v = torch.randn(M, K, generator=g, dtype=F.F64, device="cuda")
    size = torch.exp2(4 * (torch.rand(-(-M // rows), -(-K // F.BLOCK), generator=g, dtype=F.F64, device="cuda") - 0.5))
    q, e = F.quantize(v * F.spread(size, rows, M, K), rows)
    return q.float().to(fp8.E4M3), (e + 127).to(torch.uint8).view(fp8.E8M0)


def sum_error(K):
    """The stated error of the 32-bit sums, relative to the result's norm: 3e-8 for every 128 of K, beside the roundings of the
    parts' sum and the output. (A cut of a running sum loses half a last place in the mean, at most 2^-24 of it; the
    running sums' norms over the whole one's average 2/3: 4e-8 for each cut. Products held in 16 bits are 1e-3 off.)"""
    return 1e-7 + 3e-8 * K / 128


@pytest.mark.parametrize("M,N,K", F.LINEAR_FORMS + [(60, 300, 65536)])
def test_linear_in_every_form(M, N, K):
    x, xs = make(M, K, 1, seed=M + K)
    w, ws = make(N, K, 128, seed=N + K)
    out = fp8.linear(x, xs, w, ws, out_dtype=torch.float32)
    settle()
    check_product(x, xs, w, ws, out)
    ref = F.values(x, xs, 1) @ F.values(w, ws, 128).t()
    assert (out.double() - ref).norm() <= sum_error(K) * ref.norm()
    for dtype in (torch.bfloat16, torch.float16):  # the same sums, rounded once
        assert torch.equal(fp8.linear(x, xs, w, ws, out_dtype=dtype), out.to(dtype))
    settle()


@pytest.mark.parametrize("M,N,K", [(2048, 2048, 16384), (2048, 2048, 65536), (23, 4096, 16384), (8, 4096, 65536)])
def test_error_of_the_deepest_sums(M, N, K):
    """Grows with the 128s of K that one accumulator takes: all of them in a pair, a part where CTAs share a tile along K."""
    x, xs = make(M, K, 1, seed=3)
    w, ws = make(N, K, 128, seed=7)
    out = fp8.linear(x, xs, w, ws, out_dtype=torch.float32)
    settle()
    ref = F.values(x, xs, 1) @ F.values(w, ws, 128).t()
    assert (out.double() - ref).norm() <= (1e-7 + 4e-8 * plan(M, N, K, 0)["kb_split"]) * ref.norm()


def check_codes(x, xs, g, gs, u, us, q, s):
    """How many e4m3 values are not the rounded 64-bit result's. A product off by d times the products' norm turns a value whose
    product is t times that norm with a probability of at most 32 d / t (twice the relative error over e4m3's step of at
    least 2^-4 of the value); over normal products that is 32 d times 0.8 ln(1 / 32 d), 2.7e-4 for d = 1e-6, for gate
    and for up. Products held in 16 bits turn percents."""
    K = x.shape[1]
    gate, up = F.product(x, xs, g, gs)[0], F.product(x, xs, u, us)[0]
    want, e = F.quantize(gate * torch.sigmoid(gate) * up, 1)
    same = F.exponent_of(s) == e
    share = 1e-3 * max(1.0, sum_error(K) / 1e-6)
    assert (~same).sum() <= 1 + share * same.numel()
    turned = (q.float().double() != want) & F.spread(same, 1, *q.shape)
    assert turned.sum() <= 1 + share * q.numel()


@pytest.mark.parametrize("M,N,K", F.SWIGLU_FORMS)
def test_swiglu_in_every_form(M, N, K):
    x, xs = make(M, K, 1, seed=M + K)
    g, gs = make(N, K, 128, seed=N + K)
    u, us = make(N, K, 128, seed=N + K + 1)
    down = int(round(0.5 * math.log2(K)))  # gates of a few units
    gs, us = ((t.view(torch.uint8) - down).view(fp8.E8M0) for t in (gs, us))
    q, s = fp8.linear_swiglu(x, xs, g, gs, u, us)
    settle()
    check_swiglu(x, xs, g, gs, u, us, q, s)
    check_codes(x, xs, g, gs, u, us, q, s)


@pytest.mark.parametrize("tokens", [1, 100, 777])
def test_an_mlp_against_its_64_bit_chain(tokens):
    """Norm, gate/up and down against the chain in 64 bits on the same weights without any rounding of activations. An e4m3
    value is off by 2.7 % of itself in the mean square (half a step over its value is 2^-4 / m for a fraction m in [1, 2),
    uniform below that): that much in gate and in up from the norm's values, together 4.5 % of gate/up's result with silu's
    slope of up to 1.1 beside its value's, 2.7 % more from its own rounding: 5.3 % of the output's norm. Twice that is the limit."""
    weights, x, r, nw = layer(tokens, 4096, 11008, seed=tokens)
    (g, gs), (u, us), (d, ds) = weights
    out, h, _ = mlp(weights, x, r, nw)
    settle()
    h64, y = F.norm(x, r, nw, 1e-6)
    gate, up = (y @ F.values(t, ts, 128).t() for t, ts in ((g, gs), (u, us)))
    ref = (gate * torch.sigmoid(gate) * up) @ F.values(d, ds, 128).t()
    assert torch.equal(h, (x.float() + r.float()).bfloat16())
    assert (out.double() - ref).norm() <= 0.106 * ref.norm()


# ---------------------------------------------------------------- int8 norm, values that are not finite
@pytest.mark.parametrize("M", [4, 400])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_norm_to_int8_of_what_is_not_finite(M, dtype):
    """A NaN makes its row's root NaN, and NaN has no int8: the row is 0. An infinity makes the root 0, so the finite values
    are 0, and 0 * inf = NaN is 0 as well. Other rows are as they would be."""
    g = torch.Generator().manual_seed(5)
    x = torch.randn(M, 512, generator=g).to(dtype).cuda()
    w = torch.randn(512, generator=g).to(dtype).cuda()
    want, _, _ = fp8.rmsnorm_quant(x, w, position=4)
    x[0] = 0
    x[1, 7] = math.nan
    x[2, 9] = math.inf
    x[3, 0], x[3, 1] = -math.inf, math.nan
    q, s, h = fp8.rmsnorm_quant(x, w, position=4)
    qr, _, h = fp8.rmsnorm_quant(x, w, position=4, residual=torch.zeros_like(x))
    settle()
    assert s is None and (q[:4] == 0).all() and torch.equal(q[4:], want[4:]) and torch.equal(q, qr)
    assert torch.equal(torch.nan_to_num(h, nan=7.0), torch.nan_to_num(x, nan=7.0))  # the residual stream keeps them


# ---------------------------------------------------------------- chains of int8 products
def test_norms_and_gemvs_in_turn_on_the_same_buffers():
    """Two activation buffers written in turn by an int8 norm and by the GEMVs behind it, launched without a wait and in a graph: each reads
    what the kernel before it wrote, not what lay there a step earlier."""
    import ctypes as C

    import numpy as np

    import ixb_oracle as O
    from ignite_xdna_b200 import _lib as L
    K, steps, lib = 1024, 12, L.load()
    rng = np.random.default_rng(4)
    nw = torch.ones(K, dtype=torch.bfloat16, device="cuda")
    layers = []
    for _ in range(3):
        w4 = O.pack_int4(rng.integers(-8, 8, size=(K, K), dtype=np.int8))
        gpos = (5 + rng.integers(0, 4, size=(K // 128, K))).astype(np.int8)
        shift = rng.integers(9, 12, size=K).astype(np.int32)
        nbytes = C.c_uint64()
        L.check(lib.ixb_w4a8_image_bytes(K, K, C.byref(nbytes)))
        img = torch.empty(nbytes.value, dtype=torch.uint8, device="cuda")
        dw, dg, ds = (torch.from_numpy(v).cuda() for v in (w4, gpos, shift))
        L.check(lib.ixb_w4a8_prepare(dw.data_ptr(), dg.data_ptr(), K, K, img.data_ptr(), None))
        layers.append((img, ds, w4, gpos, shift))
    torch.cuda.synchronize()
    xs = [torch.randn(1, K, device="cuda").bfloat16() for _ in range(steps)]
    bufs = [torch.zeros(1, K, dtype=torch.int8, device="cuda") for _ in range(2)]
    kept = torch.zeros(steps, K, dtype=torch.int8, device="cuda")

    def chain(stream):
        for i, x in enumerate(xs):
            L.check(lib.ixb_rmsnorm_quant(x.data_ptr(), K, None, 0, nw.data_ptr(), L.BF16, L.BF16, 1, K, 1e-6, 5, None, 0,
                                          bufs[0].data_ptr(), K, None, 0, stream))
            for j, (img, ds, *_) in enumerate(layers):
                to = kept[i] if j == 2 else bufs[1 - j % 2]
                L.check(lib.ixb_w4a8_gemv(bufs[j % 2].data_ptr(), img.data_ptr(), ds.data_ptr(), to.data_ptr(), K, K, stream))

    want = []
    for x in xs:
        a = fp8.rmsnorm_quant(x, nw, position=5)[0].cpu().numpy()
        for _, _, w4, gpos, shift in layers:
            a = O.w4a8_srs(a, w4, gpos, shift)
        want.append(a[0])
    want = torch.from_numpy(np.stack(want))
    chain(torch.cuda.current_stream().cuda_stream)
    settle()
    assert torch.equal(kept.cpu(), want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        chain(torch.cuda.current_stream().cuda_stream)
    for _ in range(5):
        kept.zero_()
        graph.replay()
        settle()
        assert torch.equal(kept.cpu(), want)
    assert len(set(map(bytes, want.numpy()))) == steps and (want != 0).any()


# ---------------------------------------------------------------- two streams
def test_clusters_of_several_launches_on_two_streams():
    """Products whose CTAs wait for one another, in both forms, at once on three streams: gate/up with the widest few-token tiles, a small
    product that leaves shared memory free, a pair product. Every launch gets its TMEM, and the same bits as alone."""
    def problem(M, N, K, swiglu):
        x, xs = make(M, K, 1, M + K)
        w, ws = make(N, K, 128, N)
        if not swiglu:
            return lambda: [fp8.linear(x, xs, w, ws)]
        u, us = make(N, K, 128, N + 1)
        return lambda: list(fp8.linear_swiglu(x, xs, w, ws, u, us))

    calls = [problem(120, 3664, 12880, True), problem(32, 4096, 2048, False), problem(700, 2048, 512, False)]
    want = [c() for c in calls]
    settle()
    streams = [torch.cuda.Stream() for _ in calls]
    for turn in range(6):
        got = [[] for _ in calls]
        for _ in range(10):
            for i, st in enumerate(streams):
                with torch.cuda.stream(st):
                    got[i].append(calls[(i + turn) % 3]())
        settle()
        for i, outs in enumerate(got):
            assert all(same_bits(a, b) for o in outs for a, b in zip(o, want[(i + turn) % 3]))


# ---------------------------------------------------------------- offsets past 32 bits
def rows_in_turn(M, K, dtype, seed):
    """[M, K] of 4099 different rows, so that neighbouring tiles differ and no row has the same place in its tile twice in turn."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    some = torch.randn(4099, K, generator=g, device="cuda").to(dtype)
    return some[torch.arange(M, device="cuda") % 4099]


def test_row_operators_past_32_bit_offsets():
    """More than 2^31 values: every row as the same row of a small call."""
    M, K = 540_000, 4096
    x = rows_in_turn(M, K, torch.bfloat16, 1)
    nw = torch.randn(K, device="cuda").bfloat16()
    small = x[:4099].clone()

    def check(big, want):
        settle()
        for b, w in zip(big, want):
            b, w = b.view(torch.uint8), w.view(torch.uint8)
            for at in range(0, M, 4099):
                part = b[at:at + 4099]
                assert torch.equal(part, w[:len(part)]), at

    want = fp8.quantize(small)
    check(fp8.quantize(x), want)
    want = fp8.rmsnorm_quant(small, nw, residual=small)
    check(fp8.rmsnorm_quant(x, nw, residual=x), want)
    del x
    x = rows_in_turn(4_200_000, 528, torch.bfloat16, 2)
    q, s = fp8.quantize(x, block_rows=128)
    settle()
    last = 32_812 * 128  # the last whole blocks and the short one behind them
    for at in (0, last - 4096, 4_200_000 // 128 * 128 - 256):
        qp, sp = fp8.quantize(x[at:at + 4096], block_rows=128)
        settle()
        assert same_bits(q[at:at + 4096], qp) and same_bits(s[at // 128:at // 128 + len(sp)], sp)


@pytest.mark.parametrize("M,N,K", [(135_000, 16400, 128), (1_100_000, 144, 2064)])
def test_products_past_32_bit_offsets(M, N, K):
    """More than 2^31 outputs, and more than 2^31 bytes of x: the rows at both ends against the 64-bit form."""
    x, xs = fp8.quantize(rows_in_turn(M, K, torch.bfloat16, 3))
    w, ws = make(N, K, 128, 4)
    out = fp8.linear(x, xs, w, ws)
    settle()
    ends = (slice(0, 300), slice(M // 2, M // 2 + 300), slice(M - 300, M))
    for rows in ends:
        check_product(x[rows], xs[rows], w, ws, out[rows])
    del out
    N = N // 16 * 16
    u, us = make(N, K, 128, 5)
    w, ws = w[:N], ws[:-(-N // 128)]
    down = int(round(0.5 * math.log2(K)))
    ws, us = ((t.view(torch.uint8) - down).view(fp8.E8M0) for t in (ws, us))
    q, s = fp8.linear_swiglu(x, xs, w, ws, u, us)
    settle()
    for rows in ends:
        check_swiglu(x[rows], xs[rows], w, ws, u, us, q[rows], s[rows])
