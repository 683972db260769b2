"""fp8 linears of a decoder layer on CUDA tensors: the quantiser, the norm that feeds them, the product
and the gate/up product (``ixb_fp8_*`` and ``ixb_rmsnorm_quant`` of include/ixb200.h).

Values are ``torch.float8_e4m3fn``; scales are powers of two, ``torch.float8_e8m0fnu``, one per 128
consecutive values of an activation row, ``[M, ceil(K / 128)]``, and one per 128 x 128 block of a weight,
``[ceil(N / 128), ceil(K / 128)]``::

    wq, ws = fp8.quantize(weight, block_rows=128)                  # once
    q, s, h = fp8.rmsnorm_quant(x, norm_weight, residual=h)        # h: the new residual stream
    q, s = fp8.linear_swiglu(q, s, gate_q, gate_s, up_q, up_s)     # silu(gate) * up, quantised
    y = fp8.linear(q, s, down_q, down_s)                           # bf16

Matrices are two-dimensional, their rows contiguous, 16-byte aligned and a multiple of 16 bytes apart;
widths are multiples of 16. Calls are enqueued on the current stream of the tensors' device and return
before the kernels finish; they can be captured into a CUDA graph. Without the compiled library or a
GPU they raise: there is no fallback. They are for inference: under grad mode an input that requires grad is
refused, for there is no backward pass, and so is one with a forward-mode tangent.
"""
from __future__ import annotations

import ctypes as C
import importlib.machinery
import importlib.util
from pathlib import Path

import torch

from . import _lib as L

BLOCK = 128
E4M3 = torch.float8_e4m3fn
E8M0 = torch.float8_e8m0fnu
BINDING_PATH = Path(__file__).resolve().parent / "_ixb_torch.so"

_native = None


def _load():
    """The native binding, bound to the loaded library; raises if it was not built."""
    global _native
    if _native is None:
        lib = L.load()
        if not BINDING_PATH.exists():
            raise ImportError(f"{BINDING_PATH} is missing: build the extensions first (ignite_xdna_b200.build)")
        loader = importlib.machinery.ExtensionFileLoader("_ixb_torch", str(BINDING_PATH))
        module = importlib.util.module_from_spec(importlib.util.spec_from_file_location("_ixb_torch", BINDING_PATH, loader=loader))
        loader.exec_module(module)
        module.bind(L.IxbError, torch.OutOfMemoryError, *[C.cast(f, C.c_void_p).value for f in (
            lib.ixb_last_error, lib.ixb_fp8_quantize, lib.ixb_rmsnorm_quant, lib.ixb_fp8_linear, lib.ixb_fp8_linear_swiglu)])
        _native = module
    return _native


def quantize(x, block_rows: int = 1):
    """``(q, scale)`` of a bf16, fp16 or fp32 matrix: e4m3 with a scale per 1 x 128 values
    (``block_rows=1``, activations) or per 128 x 128 (``block_rows=128``, weights). A scale is the
    least power of two, 2**-127 at the least, that brings its block's largest finite value to 448 or
    less; rounding is to nearest even; infinities and NaN become NaN."""
    return (_native or _load()).quantize(x, block_rows)


def rmsnorm_quant(x, weight, eps: float = 1e-6, residual=None, position=None):
    """``(q, scale, h)``: y = (x + residual) / sqrt(mean((x + residual)**2) + eps) * weight in fp32,
    quantised per 1 x 128 as :func:`quantize` does; with ``position`` p, ``q`` is int8,
    clamp(rne(y * 2**p), -128, 127), what the W4A8 and int8 products read, and ``scale`` is None.
    ``h`` is x + residual rounded to x's type (a new tensor), None without a residual; the norm reads the
    unrounded sum. ``weight`` has x's type or fp32; rows hold at most 32768 values, and the products h * weight
    have to stay in fp32's range. A row with a NaN is NaN in e4m3 and 0 in int8, which has no NaN; in a row with an
    infinity the finite values are 0 and the infinity is NaN, or 0 in int8. ``h`` keeps what is not finite."""
    return (_native or _load()).rmsnorm_quant(x, weight, eps, residual, position)


def linear(x, x_scale, w, w_scale, out_dtype=torch.bfloat16, out=None):
    """``x @ w.T`` of e4m3 matrices with their scales: x ``[M, K]``, w ``[N, K]`` -> ``[M, N]`` in bf16, fp16
    or fp32, summed in fp32 by the tensor cores, which cut towards zero where an fp32 adder rounds: 2e-8 to 3e-8 of
    the result's norm for every 128 of K that one accumulator takes (many tokens: all of K, 6e-7 at 4096, 2e-6 at
    11008, 1.7e-5 at 65536, the most; few tokens: a part of K, 1e-7, 2e-7 and 1.3e-6). ``out``: a matrix of that shape to write, of any of the three types (``out_dtype`` is then not
    read), its rows contiguous, that shares no memory with the inputs: one that does is refused, and so is one that only
    meets an input's span without sharing a byte, where the two have rows of different pitch."""
    return (_native or _load()).linear(x, x_scale, w, w_scale, out_dtype, out)


def linear_swiglu(x, x_scale, gate, gate_scale, up, up_scale):
    """``(q, scale)`` of silu(x @ gate.T) * (x @ up.T): x ``[M, K]``, gate and up ``[N, K]`` (two matrices, or
    views of one, each with its own block scales) -> e4m3 ``[M, N]`` with a scale per 128 outputs of a
    row, the next :func:`linear`'s x. The products stay in fp32 inside the kernel, summed as :func:`linear`'s, so
    a value within their error of a border between two e4m3 values may fall on either side."""
    return (_native or _load()).linear_swiglu(x, x_scale, gate, gate_scale, up, up_scale)
