"""What is measured of the fp8 operators of a decoder layer's linears: their cases, inputs, plain forms and
64-bit values.

  quantize   values -> e4m3 with a power-of-two scale for each block of 128 (1 x 128, or 128 x 128 of a weight)
  norm       residual addition + root-mean-square norm -> e4m3 with scales, or int8 at a power-of-two position
  linear     e4m3 x e4m3 with the blocks' scales -> bf16, fp16 or fp32
  swiglu     two such products (gate and up), silu(gate) * up -> e4m3 with scales

`own` chooses between the plain forms (elementary torch operations in 32 bits) and the package's kernels.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BLOCK = 128      # values along a row that share a scale
E4M3_MAX = 448.0
EPS = 1e-5


def listed():
    return [
        # the attention's output on its way into the output projection, a prefill chunk of 512 tokens
        {"name": "quantize 512x4096 bf16", "op": "quantize", "rows": 1, "M": 512, "K": 4096, "dtype": "bf16"},
        # a projection's weight as it is loaded, 128 x 128 blocks; the sizes of the W4A8 bench's gate projection
        {"name": "quantize weight 11008x4096", "op": "quantize", "rows": 128, "M": 11008, "K": 4096, "dtype": "bf16"},
        # the norm before a projection at one decoded token: latency alone
        {"name": "norm 1x4096 bf16", "op": "norm", "M": 1, "K": 4096, "dtype": "bf16", "residual": True, "position": -1},
        # the same over a long prompt
        {"name": "norm 8192x4096 bf16", "op": "norm", "M": 8192, "K": 4096, "dtype": "bf16", "residual": True, "position": -1},
        # the int8 form, which the W4A8 and int8 products read, at an odd number of rows and a ragged width
        {"name": "norm 1333x5136 fp16 int8", "op": "norm", "M": 1333, "K": 5136, "dtype": "fp16", "residual": False, "position": 4},
        # one decoded token through a square projection (attention's output)
        {"name": "linear 1x4096x4096", "op": "linear", "M": 1, "N": 4096, "K": 4096, "dtype": "bf16"},
        # a decode batch of odd size through the down projection
        {"name": "linear 23x4096x11008 fp16", "op": "linear", "M": 23, "N": 4096, "K": 11008, "dtype": "fp16"},
        # a prefill chunk through the down projection
        {"name": "linear 512x4096x11008", "op": "linear", "M": 512, "N": 4096, "K": 11008, "dtype": "bf16"},
        # a ragged prompt, an output width and a depth that fill no tile
        {"name": "linear 1537x5003x2064 fp16", "op": "linear", "M": 1537, "N": 5003, "K": 2064, "dtype": "fp16"},
        # a long prompt through a wide projection: the largest product
        {"name": "linear 8192x11008x4096", "op": "linear", "M": 8192, "N": 11008, "K": 4096, "dtype": "bf16"},
        # gate and up of one decode batch
        {"name": "swiglu 8x11008x4096", "op": "swiglu", "M": 8, "N": 11008, "K": 4096, "dtype": "bf16"},
        # gate and up of a prompt
        {"name": "swiglu 2048x11008x4096", "op": "swiglu", "M": 2048, "N": 11008, "K": 4096, "dtype": "bf16"},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _width(rng, low, high):
    return 16 * _log(rng, low // 16, high // 16)


def draw(rng):
    op = rng.choice(("quantize", "norm", "linear", "linear", "swiglu"))
    case = {"op": op, "dtype": rng.choice(("bf16", "fp16"))}
    if op == "quantize":
        rows = rng.choice((1, 128))
        M, K = _log(rng, 1 if rows == 1 else 100, 11008), _width(rng, 128, 16384)
        return {**case, "rows": rows, "M": min(M, 11008 * 4096 // K), "K": K}
    if op == "norm":
        K = _width(rng, 256, 16384)
        residual, position = rng.random() < 0.7, rng.choice((-1, -1, 3, 4))
        return {**case, "M": min(_log(rng, 1, 8192), 8192 * 4096 // K), "K": K, "residual": residual, "position": position}
    M, K = _log(rng, 1, 8192), _width(rng, 256, 16384)
    if op == "linear":
        return {**case, "M": M, "K": K, "N": min(_log(rng, 64, 16384), 8192 * 11008 * 4096 // (M * K) or 1)}
    return {**case, "M": M, "K": K, "N": min(_width(rng, 128, 11008), 16 * (8192 * 5504 * 4096 // (M * K) // 16) or 16)}


def _round_blocks(v, rows):
    """v as (e4m3, e8m0 scales), each scale the least power of two that brings its block's largest value to 448 or less."""
    M, K = v.shape
    mb, kb = -(-M // rows), -(-K // BLOCK)
    p = torch.nn.functional.pad(v, (0, kb * BLOCK - K, 0, mb * rows - M)).view(mb, rows, kb, BLOCK)
    top = torch.where(torch.isfinite(p), p.abs(), 0.0).amax(dim=(1, 3), keepdim=True)
    f, k = torch.frexp(top)  # top = f * 2**k, and 448 = 0.875 * 2**9
    e = torch.where(top > 0, (k - 9 + (f > 0.875)).clamp(min=-127), -127)
    q = torch.ldexp(torch.where(torch.isfinite(p), p, math.nan), -e).to(torch.float8_e4m3fn)
    q = q.view(mb * rows, kb * BLOCK)[:M, :K].contiguous()
    return q, (e.view(mb, kb) + 127).to(torch.uint8).view(torch.float8_e8m0fnu)


def _values(q, s, rows, dtype):
    """The values that (e4m3, scales) stand for."""
    M, K = q.shape
    e = s.view(torch.uint8).to(torch.int32) - 127
    e = e.repeat_interleave(rows, 0)[:M].repeat_interleave(BLOCK, 1)[:, :K]
    return torch.ldexp(q.to(dtype), e)


def _activations(g, M, K):
    """Rows as a decoder layer has them: rows of different sizes, and a few channels far above the others."""
    x = torch.randn(M, K, device="cuda", generator=g)
    channel = torch.exp(0.5 * torch.randn(K, device="cuda", generator=g))
    channel = torch.where(torch.rand(K, device="cuda", generator=g) < 0.004, 20 * channel, channel)
    return x * channel * torch.exp(0.3 * torch.randn(M, 1, device="cuda", generator=g))


def _weight(g, N, K):
    return torch.randn(N, K, device="cuda", generator=g) * (K ** -0.5)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    op, M, K, dtype = case["op"], case["M"], case["K"], DTYPES[case["dtype"]]
    state = {"op": op, "dtype": dtype}
    if op == "quantize":
        x = _activations(g, M, K) if case["rows"] == 1 else _weight(g, M, K)
        return {**state, "x": x.to(dtype), "rows": case["rows"]}
    if op == "norm":
        state["x"] = _activations(g, M, K).to(dtype)
        state["residual"] = (2 * _activations(g, M, K)).to(dtype) if case["residual"] else None
        state["weight"] = (1 + 0.2 * torch.randn(K, device="cuda", generator=g)).to(dtype)
        state["position"] = case["position"] if case["position"] >= 0 else None
        return state
    state["x"] = _round_blocks(_activations(g, M, K), 1)
    state["w"] = _round_blocks(_weight(g, case["N"], K), 128)
    if op == "swiglu":
        state["up"] = _round_blocks(_weight(g, case["N"], K), 128)
    return state


def _product(x, w):
    return _values(*x, 1, torch.float32) @ _values(*w, 128, torch.float32).t()


def run(state):
    if own:
        return _run_own(state)
    op = state["op"]
    if op == "quantize":
        return _round_blocks(state["x"].float(), state["rows"])
    if op == "norm":
        h = state["x"].float()
        if state["residual"] is not None:
            h = h + state["residual"].float()
        y = h * torch.rsqrt(h.square().mean(1, keepdim=True) + EPS) * state["weight"].float()
        kept = [h.to(state["dtype"])] if state["residual"] is not None else []
        if state["position"] is None:
            return [*_round_blocks(y, 1), *kept]
        # an int8 q at position p stands for q / 2**p, which fp16 holds exactly
        q = torch.round(y * 2.0 ** state["position"]).clamp(-128, 127)
        return [(q * 2.0 ** -state["position"]).half(), *kept]
    if op == "linear":
        return _product(state["x"], state["w"]).to(state["dtype"])
    gate = _product(state["x"], state["w"])
    return _round_blocks(gate / (1 + torch.exp(-gate)) * _product(state["x"], state["up"]), 1)


def _run_own(state):
    from ignite_xdna_b200 import fp8
    op = state["op"]
    if op == "quantize":
        return fp8.quantize(state["x"], block_rows=state["rows"])
    if op == "norm":
        q, scale, h = fp8.rmsnorm_quant(state["x"], state["weight"], eps=EPS, residual=state["residual"],
                                        position=state["position"])
        kept = [h] if h is not None else []
        if scale is None:
            return [q.half() * 2.0 ** -state["position"], *kept]
        return [q, scale, *kept]
    if op == "linear":
        return fp8.linear(*state["x"], *state["w"], out_dtype=state["dtype"])
    return fp8.linear_swiglu(*state["x"], *state["w"], *state["up"])


def work(case):
    op, M, K = case["op"], case["M"], case["K"]
    size = torch.empty((), dtype=DTYPES[case["dtype"]]).element_size()
    kb = -(-K // BLOCK)
    if op == "quantize":
        return {"bytes": M * K * (size + 1) + -(-M // case["rows"]) * kb, "flops": 2 * M * K}
    if op == "norm":
        # x read and the 8-bit values written; the residual read and the new one written
        scales = M * kb if case["position"] < 0 else 0
        return {"bytes": M * K * (size + 1 + 2 * size * case["residual"]) + scales + K * size, "flops": 6 * M * K}
    N = case["N"]
    if op == "linear":
        return {"bytes": M * (K + kb) + N * K + -(-N // 128) * kb + M * N * size, "flops": 2 * M * N * K}
    return {"bytes": M * (K + kb) + 2 * (N * K + -(-N // 128) * kb) + M * (N + -(-N // BLOCK)),
            "flops": 4 * M * N * K + 8 * M * N}


def _exact_blocks(y, rows):
    """The nearest e4m3 values and their scales of 64-bit y, from the definition: 3 fraction bits down to 2**-6, steps of 2**-9 below."""
    M, K = y.shape
    mb, kb = -(-M // rows), -(-K // BLOCK)
    wide = torch.zeros(mb * rows, kb * BLOCK, dtype=torch.float64, device=y.device)
    wide[:M, :K] = y
    top = wide.abs().view(mb, rows, kb, BLOCK).transpose(1, 2).reshape(mb, kb, -1).max(2).values
    e = torch.ceil(torch.log2(top / E4M3_MAX).clamp(-127, 127))
    # the logarithm may be off next to a power of two: one up, or one down where that still holds the largest value
    e = e + (torch.exp2(e) * E4M3_MAX < top).double() - ((torch.exp2(e - 1) * E4M3_MAX >= top) & (e > -127)).double()
    v = y / torch.exp2(e).repeat_interleave(rows, 0)[:M].repeat_interleave(BLOCK, 1)[:, :K]
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6))) - 3)
    return [torch.round(v / step) * step, torch.exp2(e)]


def _exact_product(x, w):
    (a, sa), (b, sb) = x, w
    sa = torch.exp2(sa.view(torch.uint8).double() - 127)
    sb = torch.exp2(sb.view(torch.uint8).double() - 127)
    K = a.shape[1]
    col = torch.arange(K, device=a.device) // BLOCK
    a64 = a.double() * sa[:, col]
    b64 = b.double() * sb[torch.arange(b.shape[0], device=b.device) // 128][:, col]
    return torch.matmul(a64, b64.transpose(0, 1))


def exact(case, seed):
    state = prepare(case, seed)
    if state["op"] == "quantize":
        return _exact_blocks(state["x"].double(), state["rows"])
    if state["op"] == "norm":
        h = state["x"].double()
        if state["residual"] is not None:
            h += state["residual"].double()
        y = h / torch.sqrt((h ** 2).sum(1) / case["K"] + EPS)[:, None] * state["weight"].double()[None]
        kept = [h] if state["residual"] is not None else []
        if state["position"] is None:
            return [*_exact_blocks(y, 1), *kept]
        unit = 2.0 ** -state["position"]
        return [torch.clamp(torch.round(y / unit), -128, 127) * unit, *kept]
    if state["op"] == "linear":
        return _exact_product(state["x"], state["w"])
    gate = _exact_product(state["x"], state["w"])
    return _exact_blocks(gate * torch.sigmoid(gate) * _exact_product(state["x"], state["up"]), 1)
