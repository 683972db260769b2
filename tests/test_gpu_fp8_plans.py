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
