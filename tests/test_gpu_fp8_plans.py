"""The fp8 products in every form that the planner picks, at a decoder's depths: chains of launches, scale images
that follow one another, accuracy of the 32-bit sums."""
import pytest
import torch

import fp8_model as F
from ignite_xdna_b200 import fp8
from test_gpu_fp8 import same_bits, settle

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
