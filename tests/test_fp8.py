"""The fp8 linears without a GPU: launch plans fit the hardware, arguments are refused before any CUDA
call, and the 64-bit forms the GPU tests compare with agree with torch's e4m3."""
import ctypes as C

import pytest
import torch

import fp8_model as F
from ignite_xdna_b200 import _lib as L
from ignite_xdna_b200 import fp8

FIELDS = ("cg", "mt", "bn", "n_tiles", "m_tiles", "kblocks", "split", "kb_split", "stages", "grid", "smem", "tmem", "nacc")


def plan(M, N, K, swiglu):
    info = (C.c_int32 * 13)()
    L.check(L.load().ixb_fp8_plan_info(M, N, K, swiglu, info, 13))
    return dict(zip(FIELDS, info))


@pytest.mark.parametrize("swiglu", [0, 1])
def test_plans_fit_the_hardware(swiglu):
    sizes = [1, 2, 15, 16, 17, 23, 33, 64, 100, 127, 128, 129, 240, 241, 256, 257, 512, 1000, 1537, 2048, 8192, 70000]
    depths = [16, 128, 144, 256, 512, 528, 2064, 4096, 11008, 16384]
    for M in sizes:
        for N in [16, 64, 128, 144, 512, 2064, 4096, 11008, 32768]:
            for K in depths:
                p = plan(M, N, K, swiglu)
                groups = -(-p["bn"] // 128)
                assert p["bn"] % 16 == 0 and 16 <= p["bn"] <= 256 and p["mt"] in (1, 2)
                assert p["cg"] in (1, 2) and p["bn"] % (16 * p["cg"]) == 0 and (p["cg"] == 1 or p["split"] == 1)
                assert p["m_tiles"] * p["bn"] >= M and p["n_tiles"] * 128 * (1 if swiglu else p["cg"] * p["mt"]) >= N
                assert p["kblocks"] * 128 >= K and p["stages"] >= 1 and p["smem"] <= 227 * 1024
                assert p["nacc"] * p["mt"] * p["bn"] + 8 * (p["mt"] + groups) <= p["tmem"] <= 512
                assert p["tmem"] & (p["tmem"] - 1) == 0
                # every CTA of a cluster has K-blocks of its own, and together they have all
                assert (p["split"] - 1) * p["kb_split"] < p["kblocks"] <= p["split"] * p["kb_split"]
                tiles = p["n_tiles"] * p["m_tiles"]
                assert p["grid"] == tiles * p["split"] if p["cg"] == 1 else 2 <= p["grid"] <= min(2 * tiles, 148)
                if p["cg"] == 1:  # the parts to add fit where the operands were
                    assert p["mt"] * p["bn"] * 512 <= p["stages"] * (p["mt"] * 16384 + p["bn"] * 128)


def test_plan_refuses_bad_sizes():
    info = (C.c_int32 * 13)()
    lib = L.load()
    for M, N, K in [(0, 16, 16), (-1, 16, 16), ((1 << 30) + 1, 16, 16), (16, 0, 16), (16, 16, 8), (16, 16, 24), (16, 16, 0), (1, 1 << 25, 16),
                    (1, 16, 65552)]:
        assert lib.ixb_fp8_plan_info(M, N, K, 0, info, 13) == L.IXB_ERR_INVALID, (M, N, K)
    assert lib.ixb_fp8_plan_info(16, 16, 16, 0, info, 12) == L.IXB_ERR_INVALID


P, ODD = 4096, 4104  # pointers that are never followed: every call below is refused on the host


@pytest.mark.parametrize("change,needle", [
    ({"x": None}, "null"), ({"xs": None}, "null"), ({"w": None}, "null"), ({"ws": None}, "null"), ({"out": None}, "out"),
    ({"x": ODD}, "aligned"), ({"w": ODD}, "aligned"), ({"ldx": 264}, "stride"), ({"ldx": 128}, "stride"),
    ({"ldw": 240}, "stride"), ({"ldxs": 1}, "scales"), ({"ldws": 1}, "scales"), ({"out": 4097}, "aligned"),
    ({"ldo": 63}, "stride"), ({"type": 3}, "type"), ({"type": -1}, "type"), ({"M": -1}, "M >= 0"), ({"N": 0}, "N in"),
    ({"K": 250}, "multiple of 16"), ({"K": 0}, "multiple of 16"),
])
def test_linear_refuses(change, needle):
    a = {"x": P, "ldx": 256, "xs": P, "ldxs": 2, "w": P, "ldw": 256, "ws": P, "ldws": 2, "out": P, "type": L.BF16,
         "ldo": 64, "M": 4, "N": 64, "K": 256, **change}
    lib = L.load()
    assert lib.ixb_fp8_linear(*a.values(), None) == L.IXB_ERR_INVALID
    assert needle in lib.ixb_last_error().decode()


@pytest.mark.parametrize("change,needle", [
    ({"N": 72}, "multiple of 16"), ({"up": None}, "null up"), ({"g": ODD}, "gate"), ({"q": None}, "null q"),
    ({"ldq": 72}, "q must"), ({"ldq": 48}, "q must"), ({"lds": 0}, "q scales"), ({"ldus": 1}, "up scales"),
])
def test_swiglu_refuses(change, needle):
    a = {"x": P, "ldx": 256, "xs": P, "ldxs": 2, "g": P, "ldg": 256, "gs": P, "ldgs": 2, "up": P, "ldu": 256, "us": P,
         "ldus": 2, "q": P, "ldq": 64, "s": P, "lds": 1, "M": 4, "N": 64, "K": 256, **change}
    lib = L.load()
    assert lib.ixb_fp8_linear_swiglu(*a.values(), None) == L.IXB_ERR_INVALID
    assert needle in lib.ixb_last_error().decode()


@pytest.mark.parametrize("change", [
    {"x": None}, {"q": None}, {"s": None}, {"x": ODD}, {"q": ODD}, {"ldx": 260}, {"ldx": 128}, {"ldq": 200}, {"lds": 1},
    {"type": 7}, {"K": 200}, {"K": 0}, {"M": -1}, {"rows": 2}, {"rows": 0},
])
def test_quantize_refuses(change):
    a = {"x": P, "type": L.F16, "ldx": 256, "M": 4, "K": 256, "rows": 1, "q": P, "ldq": 256, "s": P, "lds": 2, **change}
    assert L.load().ixb_fp8_quantize(*a.values(), None) == L.IXB_ERR_INVALID


@pytest.mark.parametrize("change", [
    {"x": None}, {"w": None}, {"q": None}, {"x": ODD}, {"w": ODD}, {"r": ODD}, {"h": ODD}, {"q": ODD}, {"h": None}, {"r": None},
    {"ldx": 252}, {"ldr": 128}, {"ldh": 128}, {"ldq": 264}, {"lds": 1}, {"type": 5}, {"wtype": L.BF16}, {"K": 40}, {"K": 0},
    {"K": 32784}, {"M": -3}, {"eps": -1.0}, {"eps": float("inf")}, {"eps": float("nan")}, {"s": None, "position": 65},
    {"s": None, "position": -65},
])
def test_norm_refuses(change):
    a = {"x": P, "ldx": 256, "r": P, "ldr": 256, "w": P, "type": L.F16, "wtype": L.F32, "M": 4, "K": 256, "eps": 1e-6,
         "position": 0, "h": P, "ldh": 256, "q": P, "ldq": 256, "s": P, "lds": 2, **change}
    assert L.load().ixb_rmsnorm_quant(*a.values(), None) == L.IXB_ERR_INVALID


def test_no_rows_is_no_work():
    lib = L.load()
    assert lib.ixb_fp8_quantize(None, L.BF16, 16, 0, 16, 1, None, 16, None, 1, None) == 0
    assert lib.ixb_rmsnorm_quant(None, 16, None, 0, None, 0, 0, 0, 16, 1e-6, 0, None, 0, None, 16, P, 1, None) == 0
    assert lib.ixb_fp8_linear(None, 16, None, 1, None, 16, None, 1, None, 0, 16, 0, 16, 16, None) == 0
    assert lib.ixb_fp8_linear_swiglu(*[None, 16] * 8, 0, 16, 16, None) == 0


def test_python_refuses_what_is_not_a_cuda_matrix():
    x = torch.zeros(4, 256, dtype=torch.bfloat16)
    q, s = F.make(4, 256, 1, 0)
    w, ws = F.make(128, 256, 128, 1)
    with pytest.raises(ValueError, match="CUDA"):
        fp8.quantize(x)
    with pytest.raises(TypeError, match="bfloat16"):
        fp8.quantize(x.double())
    with pytest.raises(ValueError, match="CUDA"):
        fp8.rmsnorm_quant(x, x[0])
    with pytest.raises(ValueError, match="CUDA"):
        fp8.linear(q, s, w, ws)
    with pytest.raises(ValueError, match="CUDA"):
        fp8.linear_swiglu(q, s, w, ws, w, ws)
    with pytest.raises(TypeError, match="tensor"):
        fp8.linear(None, s, w, ws)
    with pytest.raises(TypeError, match="tensor"):
        fp8.quantize([1.0])
    with pytest.raises(TypeError):
        fp8.quantize(x, block_rows="many")
    with pytest.raises(ValueError, match="grad"):
        fp8.quantize(x.clone().requires_grad_())
    with pytest.raises(ValueError, match="strided"):
        fp8.quantize(x.to_sparse())


def test_the_model_rounds_as_torch_does():
    """e4m3() against torch's conversion on every e4m3 value, the midpoints between neighbours and values either side."""
    codes = torch.arange(0x7F, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    mid = (codes[1:] + codes[:-1]) / 2
    v = torch.cat([codes, mid, mid * (1 + 2.0 ** -20), mid * (1 - 2.0 ** -20)])
    v = torch.cat([v, -v])
    assert torch.equal(F.e4m3(v), v.float().to(torch.float8_e4m3fn).double())
    top = torch.tensor([[0.0, 448.0, 448.0 * 2.0 ** -140, 449.0, 3.0e38, 1.75, 1.7500001]], dtype=torch.float64)
    e = F.exponents(top)
    assert e.tolist() == [[-127.0, 0.0, -127.0, 1.0, 120.0, -8.0, -7.0]]
