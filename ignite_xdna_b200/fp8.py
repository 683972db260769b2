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
GPU they raise: there is no fallback.
"""
from __future__ import annotations

import torch

from . import _lib as L

BLOCK = 128
E4M3 = torch.float8_e4m3fn
E8M0 = torch.float8_e8m0fnu
_TYPES = {torch.bfloat16: L.BF16, torch.float16: L.F16, torch.float32: L.F32}


def _rows(t, name, dtype=None, shape=None):
    """Checks a matrix with contiguous rows; returns (pointer, row stride)."""
    if t.dim() != 2 or not t.is_cuda:
        raise ValueError(f"{name}: a two-dimensional CUDA tensor is needed, got {tuple(t.shape)} on {t.device}")
    if dtype is not None and t.dtype is not dtype:
        raise TypeError(f"{name}: {dtype} is needed, got {t.dtype}")
    if shape is not None and t.shape != shape:
        raise ValueError(f"{name}: shape {tuple(shape)} is needed, got {tuple(t.shape)}")
    rows, cols = t.shape
    ld, step = t.stride()
    if step != 1 and cols > 1:
        raise ValueError(f"{name}: the values of a row must be contiguous")
    if rows <= 1:  # the stride of a single row says nothing
        return t.data_ptr(), -(-cols // 16) * 16
    if ld < cols:
        raise ValueError(f"{name}: rows overlap (stride {ld} below {cols})")
    return t.data_ptr(), ld


def _same_device(first, *others):
    for t in others:
        if t is not None and t.device != first.device:
            raise ValueError(f"tensors on different devices: {first.device} and {t.device}")


def _call(name, device, *args):
    """The library call on `device`'s current stream."""
    lib = L.load()
    if device.index == torch.cuda.current_device():
        L.check(getattr(lib, name)(*args, torch.cuda.current_stream(device).cuda_stream))
    else:
        with torch.cuda.device(device):
            L.check(getattr(lib, name)(*args, torch.cuda.current_stream(device).cuda_stream))


def _blocks(n):
    return -(-n // BLOCK)


def _scales(rows, cols, device):
    """An empty scale matrix whose rows start on 4 bytes, which the products read a word at a time."""
    n = _blocks(cols)
    return torch.empty((rows, -(-n // 4) * 4), dtype=E8M0, device=device)[:, :n]


def quantize(x, block_rows: int = 1):
    """``(q, scale)`` of a bf16, fp16 or fp32 matrix: e4m3 with a scale per 1 x 128 values
    (``block_rows=1``, activations) or per 128 x 128 (``block_rows=128``, weights). A scale is the
    least power of two, 2**-127 at the least, that brings its block's largest finite value to 448 or
    less; rounding is to nearest even; infinities and NaN become NaN."""
    if x.dtype not in _TYPES:
        raise TypeError(f"x: bfloat16, float16 or float32 is needed, got {x.dtype}")
    px, ldx = _rows(x, "x")
    M, K = x.shape
    q = torch.empty((M, K), dtype=E4M3, device=x.device)
    scale = _scales(M if block_rows == 1 else _blocks(M), K, x.device)
    _call("ixb_fp8_quantize", x.device, px, _TYPES[x.dtype], ldx, M, K, block_rows, q.data_ptr(), K, scale.data_ptr(),
          scale.stride(0))
    return q, scale


def rmsnorm_quant(x, weight, eps: float = 1e-6, residual=None, position=None):
    """``(q, scale, h)``: y = (x + residual) / sqrt(mean((x + residual)**2) + eps) * weight in fp32,
    quantised per 1 x 128 as :func:`quantize` does; with ``position`` p, ``q`` is int8,
    clamp(rne(y * 2**p), -128, 127), what the W4A8 and int8 products read, and ``scale`` is None.
    ``h`` is x + residual rounded to x's type (a new tensor), None without a residual; the norm reads the
    unrounded sum. ``weight`` has x's type or fp32; rows hold at most 32768 values."""
    if x.dtype not in _TYPES:
        raise TypeError(f"x: bfloat16, float16 or float32 is needed, got {x.dtype}")
    px, ldx = _rows(x, "x")
    M, K = x.shape
    if weight.shape != (K,) or not weight.is_contiguous() or not weight.is_cuda:
        raise ValueError(f"weight: a contiguous CUDA tensor of {K} values is needed, got {tuple(weight.shape)} on {weight.device}")
    if weight.dtype is not x.dtype and weight.dtype is not torch.float32:
        raise TypeError(f"weight: {x.dtype} or float32 is needed, got {weight.dtype}")
    _same_device(x, weight, residual)
    pr, ldr, h = None, 0, None
    if residual is not None:
        pr, ldr = _rows(residual, "residual", x.dtype, x.shape)
        h = torch.empty((M, K), dtype=x.dtype, device=x.device)
    q = torch.empty((M, K), dtype=E4M3 if position is None else torch.int8, device=x.device)
    scale = _scales(M, K, x.device) if position is None else None
    _call("ixb_rmsnorm_quant", x.device, px, ldx, pr, ldr, weight.data_ptr(), _TYPES[x.dtype], _TYPES[weight.dtype], M, K,
          eps, 0 if position is None else position, None if h is None else h.data_ptr(), K, q.data_ptr(), K,
          None if scale is None else scale.data_ptr(), 0 if scale is None else scale.stride(0))
    return q, scale, h


def _operand(q, scale, name, rows, K):
    """Pointers and strides of an e4m3 matrix [*, K] with its scales; `rows`: rows per scale."""
    pq, ld = _rows(q, name, E4M3)
    if q.shape[1] != K:
        raise ValueError(f"{name}: {K} columns are needed, got {q.shape[1]}")
    ps, lds = _rows(scale, f"{name} scale", E8M0, (-(-q.shape[0] // rows), _blocks(K)))
    return pq, ld, ps, lds


def linear(x, x_scale, w, w_scale, out_dtype=torch.bfloat16, out=None):
    """``x @ w.T`` of e4m3 matrices with their scales: x ``[M, K]``, w ``[N, K]`` -> ``[M, N]`` in bf16, fp16
    or fp32, summed in fp32. ``out``: a matrix of that shape and type to write, its rows contiguous."""
    M, K = x.shape
    N = w.shape[0]
    ax = _operand(x, x_scale, "x", 1, K)
    aw = _operand(w, w_scale, "w", BLOCK, K)
    if out is None:
        if out_dtype not in _TYPES:
            raise TypeError(f"out_dtype: bfloat16, float16 or float32 is needed, got {out_dtype}")
        out = torch.empty((M, N), dtype=out_dtype, device=x.device)
        po, ldo = out.data_ptr(), N
    else:
        if out.dtype not in _TYPES:
            raise TypeError(f"out: bfloat16, float16 or float32 is needed, got {out.dtype}")
        po, ldo = _rows(out, "out", None, (M, N))
    _same_device(x, x_scale, w, w_scale, out)
    _call("ixb_fp8_linear", x.device, *ax, *aw, po, _TYPES[out.dtype], ldo, M, N, K)
    return out


def linear_swiglu(x, x_scale, gate, gate_scale, up, up_scale):
    """``(q, scale)`` of silu(x @ gate.T) * (x @ up.T): x ``[M, K]``, gate and up ``[N, K]`` (two matrices, or
    views of one, each with its own block scales) -> e4m3 ``[M, N]`` with a scale per 128 outputs of a
    row, the next :func:`linear`'s x. The products stay in fp32 inside the kernel."""
    M, K = x.shape
    N = gate.shape[0]
    ax = _operand(x, x_scale, "x", 1, K)
    ag = _operand(gate, gate_scale, "gate", BLOCK, K)
    au = _operand(up, up_scale, "up", BLOCK, K)
    if up.shape[0] != N:
        raise ValueError(f"gate and up have {N} and {up.shape[0]} rows")
    _same_device(x, x_scale, gate, gate_scale, up, up_scale)
    q = torch.empty((M, N), dtype=E4M3, device=x.device)
    scale = _scales(M, N, x.device)
    _call("ixb_fp8_linear_swiglu", x.device, *ax, *ag, *au, q.data_ptr(), N, scale.data_ptr(), scale.stride(0), M, N, K)
    return q, scale
