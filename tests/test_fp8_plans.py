"""The fp8 products' launch plans, without a GPU: what keeps launches on several streams from waiting for one another,
and that the GPU tests reach every form."""
import random
import re
from pathlib import Path

import pytest
import torch

import fp8_model as F
from ignite_xdna_b200 import fp8
from test_fp8 import plan

SM_SHARED, SYSTEM = 228 * 1024, 1024  # an SM's shared memory, and what the system takes of it per CTA
SIZES = [1, 7, 16, 17, 40, 64, 100, 112, 113, 120, 127, 128, 129, 240, 256, 400, 512, 1537, 4096]


@pytest.mark.parametrize("swiglu", [0, 1])
def test_clusters_cannot_wait_for_one_anothers_tmem(swiglu):
    """An allocation waits for the columns of the SM's other CTAs, and a cluster's CTAs for one another. Few tokens: two CTAs
    per SM at the most, each with at most half of TMEM. Pairs: alone on their SMs."""
    r = random.Random(1)
    depths = [16, 144, 256, 528, 2064, 4096, 11008, 12880] + [16 * r.randint(1, 1024) for _ in range(30)]
    cases = [(120, 3664, 12880)] + [(M, N, K) for M in SIZES for N in (16, 144, 1024, 3664, 11008) for K in depths]
    for M, N, K in cases:
        p = plan(M, N, K, swiglu)
        if p["cg"] == 1:
            assert p["tmem"] <= 256 and 3 * (p["smem"] + SYSTEM) > SM_SHARED, (M, N, K, p)
        else:
            assert p["tmem"] <= 512 and p["smem"] + SYSTEM == SM_SHARED, (M, N, K, p)


def kernels(name):
    """The source without comments, and its parts: from one kernel's __global__ to the next."""
    text = (Path(__file__).resolve().parent.parent / "ignite_xdna_b200" / "csrc" / name).read_text()
    text = re.sub(r"//[^\n]*|/\*.*?\*/", "", text, flags=re.S)
    return text, text.split("__global__")[1:]


def test_fp8_kernels_read_nothing_as_read_only():
    """Each of them may start while the kernel that writes its inputs runs (programmatic dependent launch), so no load
    may be one of data that is read-only for the whole kernel: no .nc load, no __ldg, and no const __restrict__ pointer,
    which lets the compiler make one."""
    text, parts = kernels("ixb_fp8.cuh")
    assert all("grid_dep_wait" in k for k in parts) and len(parts) == 4
    assert not re.search(r"\.nc\b|__ldg|__restrict__", text)


# ---------------------------------------------------------------- arguments
def places(t):
    """The bytes that a matrix takes, as a set of addresses."""
    size, row = t.element_size(), t.stride(0) * t.element_size()
    return {t.data_ptr() + i * row + j for i in range(t.shape[0]) for j in range(t.shape[1] * size)}


def test_what_shares_memory():
    """Against the sets of bytes: exact where rows are equally far apart or one matrix has one row, never 'no' for matrices
    that share a byte, never 'yes' for spans that do not meet."""
    fp8._load()
    shares = fp8._native.shares_memory
    r = random.Random(3)
    buf = torch.zeros(4096, dtype=torch.uint8)
    seen = [0, 0]
    for _ in range(4000):
        views = []
        pitch = 4 * r.randint(1, 16)
        for _ in range(2):
            t = buf.view(r.choice((torch.uint8, torch.bfloat16, torch.float32)))
            size = t.element_size()
            step = (pitch if r.random() < 0.7 else 4 * r.randint(1, 16)) // size
            rows, cols = r.randint(1, 6), r.randint(1, step)
            views.append(t.as_strided((rows, cols), (step, 1), r.randint(0, 160) // size))
        a, b = views
        pa, pb = places(a), places(b)
        got, true = shares(a, b), bool(pa & pb)
        assert got or not true
        if a.shape[0] == 1 or b.shape[0] == 1 or a.stride(0) * a.element_size() == b.stride(0) * b.element_size():
            assert got == true, (a.shape, a.stride(), a.dtype, b.shape, b.stride(), b.dtype)
            seen[true] += 1
        if max(pa) < min(pb) or max(pb) < min(pa):
            assert not got
    assert min(seen) > 200
    assert not shares(buf.view(64, 64)[:0], buf.view(64, 64))


def test_a_forward_mode_tangent_is_refused():
    import torch.autograd.forward_ad as fwd
    x = torch.zeros(4, 256)
    with fwd.dual_level():
        dual = fwd.make_dual(x, torch.ones_like(x))
        with pytest.raises(ValueError, match="tangent"):
            fp8.quantize(dual)
        with torch.no_grad(), pytest.raises(ValueError, match="tangent"):  # forward mode goes on under no_grad
            fp8.rmsnorm_quant(x, dual[0])
        with pytest.raises(ValueError, match="CUDA"):  # refused for its device alone
            fp8.quantize(fwd.unpack_dual(dual).primal)
    with pytest.raises(ValueError, match="CUDA"):
        fp8.quantize(x)


def test_a_view_of_negated_values_is_refused():
    """Its memory holds the opposite of its values, and the kernels read memory."""
    x = torch.ones(4, 256)
    with pytest.raises(ValueError, match="negated"):
        fp8.quantize(torch._neg_view(x))
    with pytest.raises(ValueError, match="negated"):
        fp8.quantize(torch.ones(4, 256, dtype=torch.complex64).conj().imag)
    with pytest.raises(ValueError, match="CUDA"):
        fp8.quantize(torch._neg_view(x).resolve_neg())


# ---------------------------------------------------------------- what the GPU tests reach
@pytest.mark.parametrize("swiglu", [0, 1])
def test_the_gpu_tests_shapes_reach_every_form(swiglu):
    shapes = F.SWIGLU_FORMS if swiglu else F.LINEAR_FORMS
    tested = {F.form(plan(*s, swiglu), swiglu) for s in shapes}
    r = random.Random(9)
    spread = lambda a, b: int(round(a * (b / a) ** r.random()))  # noqa: E731
    missing = {}
    for _ in range(10000):
        s = (spread(1, 8192), 16 * spread(1, 1024) if swiglu else spread(1, 16384), 16 * spread(1, 1024))
        missing.setdefault(F.form(plan(*s, swiglu), swiglu), s)
    missing = {f: s for f, s in missing.items() if f not in tested}
    assert not missing
    assert len(tested) >= (20 if swiglu else 34)


def test_the_gemv_reads_its_activations_as_what_another_kernel_writes():
    """It starts while the kernel before, a norm or another GEMV, may still write them."""
    _, parts = kernels("ixb_w4a8.cuh")
    gemv = next(k for k in parts if "w4a8_gemv_kernel(" in k)
    assert "grid_dep_launch" in gemv and "const int8_t* a," in gemv and "int8_t* out," in gemv
    assert not re.search(r"__ldg\((reinterpret_cast<const int4\*>\()?a\b", gemv)
