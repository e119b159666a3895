"""Feed-forward layers as a program trains and serves them, as a list of cases that can be timed and compared.

Each case is one call of a public operator of the `beam` package on torch tensors:

    gated     h = silu(a @ b[:N].T) * (a @ b[N:].T), and with "train" the pre-activations gu = a @ b.T
              beam.gemmrc_gated
    gated_bw  the gradients da [M, K] and db [2N, K] of that layer from dh, gu, a and b
              beam.gemmrc_gated_backward
    quant     x in 4-bit floating point with a power of two for every 32 elements (MXFP4), read back as the values held
              beam.mxfp4_quantize, beam.mxfp4_dequantize
    product   c = a @ b.T of two operands held in MXFP4
              beam.gemmrc_mxfp4
    linear    c = mxfp4(a) @ b.T, a in 16 bits and quantised in the call, b held in MXFP4
              beam.linear_mxfp4

`listed()` holds one representative of every range, `draw()` takes further cases out of the same ranges.

MXFP4 here: two elements to a byte, the even one in the low half, e2m1 (0, 0.5, 1, 1.5, 2, 3, 4, 6 and a sign); the power of
two of row m, block b (32 elements along K) is a biased exponent (e8m0) in scales[b // 8, m, b % 8], zero behind the last block.
"""
import os
import sys

import torch

own = False  # False: elementary torch operations in 32 bits; True: this library's operators

_DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
_LEVELS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def listed():
    return [
        # serving: one token through a wide gated layer, the weights are read once
        {"name": "gated_token", "op": "gated", "dtype": "bf16", "M": 1, "N": 11008, "K": 4096, "train": False},
        # sizes as data sets have them: no tile divides them
        {"name": "gated_ragged", "op": "gated", "dtype": "fp16", "M": 1001, "N": 2001, "K": 2000, "train": False},
        # training: thousands of tokens, pre-activations kept for the backward pass
        {"name": "gated_train", "op": "gated", "dtype": "bf16", "M": 4096, "N": 11008, "K": 4096, "train": True},
        # the backward pass of a short batch through a small layer: three launches' latency
        {"name": "gated_bw_small", "op": "gated_bw", "dtype": "fp16", "M": 512, "N": 1024, "K": 512},
        # an odd number of tokens: the sum over them has rows that start anywhere
        {"name": "gated_bw_ragged", "op": "gated_bw", "dtype": "bf16", "M": 1001, "N": 2001, "K": 2000},
        # the backward pass that goes with gated_train
        {"name": "gated_bw_train", "op": "gated_bw", "dtype": "bf16", "M": 4096, "N": 11008, "K": 4096},
        # a few tokens' activations on their way into a 4-bit product
        {"name": "quant_tokens", "op": "quant", "dtype": "bf16", "M": 16, "K": 4096},
        # a weight matrix, once, when a model is loaded
        {"name": "quant_weight", "op": "quant", "dtype": "fp16", "M": 8192, "K": 8192},
        # both operands held in 4 bits, sizes that no tile divides
        {"name": "product_ragged", "op": "product", "dtype": "fp16", "M": 1001, "N": 2001, "K": 2016},
        # the large square product that the benchmark quotes
        {"name": "product_8192", "op": "product", "dtype": "bf16", "M": 8192, "N": 8192, "K": 8192},
        # serving with 4-bit weights: one token, latency counts
        {"name": "linear_token", "op": "linear", "dtype": "bf16", "M": 1, "N": 11008, "K": 4096},
        # ... and a batch of prompts
        {"name": "linear_prompts", "op": "linear", "dtype": "bf16", "M": 2048, "N": 4096, "K": 11008},
    ]


def _log(rng, lo, hi, step=1):
    """A multiple of `step` in [lo, hi], spread evenly over its logarithm."""
    v = lo * (hi / lo) ** rng.random()
    return max(step, min(hi, int(round(v / step)) * step))


def draw(rng):
    op = rng.choice(["gated", "gated", "gated_bw", "gated_bw", "quant", "product", "linear"])
    dtype = rng.choice(["fp16", "bf16"])
    step = rng.choice([1, 8, 64])
    tokens = _log(rng, 1, 4096)
    if op == "gated":
        return {"op": op, "dtype": dtype, "M": tokens, "N": _log(rng, 64, 11008, step), "K": _log(rng, 64, 4096, step),
                "train": rng.random() < 0.5}
    if op == "gated_bw":
        return {"op": op, "dtype": dtype, "M": tokens, "N": _log(rng, 64, 11008, step), "K": _log(rng, 64, 4096, step)}
    if op == "quant":
        return {"op": op, "dtype": dtype, "M": _log(rng, 1, 8192), "K": _log(rng, 32, 8192, 32)}
    return {"op": op, "dtype": dtype, "M": _log(rng, 1, 8192), "N": _log(rng, 64, 8192, step), "K": _log(rng, 64, 8192, 32)}


# ---------------------------------------------------------------------------- plain forms


def _silu_and_slope(g):
    s = 1 / (1 + torch.exp(-g))
    return g * s, s * (1 + g * (1 - s))


def _plain_gated(a, b):
    gu = a.float() @ b.float().t()
    N = b.shape[0] // 2
    return _silu_and_slope(gu[:, :N])[0] * gu[:, N:], gu


def _plain_gated_bw(dh, gu, a, b):
    N = dh.shape[1]
    g, u, dh = gu[:, :N].float(), gu[:, N:].float(), dh.float()
    act, slope = _silu_and_slope(g)
    dgu = torch.cat((dh * u * slope, dh * act), 1)
    return dgu @ b.float(), dgu.t() @ a.float()


def _times_power(v, e):
    """v * 2^e, e whole, in two steps whose powers are normal numbers."""
    half = e // 2
    return v * ((half + 127) << 23).view(torch.float32) * ((e - half + 127) << 23).view(torch.float32)


def _plain_quant(x):
    """Codes 0 .. 15 [M, K] and biased exponents [M, K / 32] of finite values."""
    M, K = x.shape
    v = x.float().view(M, K // 32, 32)
    # the largest magnitude is in [2^(e + 2), 2^(e + 3)): up to 8 of the scale, and what lies beyond 6 becomes 6
    e = torch.frexp(v.abs().amax(2))[1] - 3
    e = torch.where(v.abs().amax(2) == 0, torch.full_like(e, -127), e).clamp(min=-127)
    y = _times_power(v, -e.unsqueeze(2)).abs()
    # nearest of the eight magnitudes, ties to the even code
    code = ((y > 0.25).int() + (y >= 0.75) + (y > 1.25) + (y >= 1.75) + (y > 2.5) + (y >= 3.5) + (y > 5))
    code = code + 8 * torch.signbit(v).int()
    return code.view(M, K), e + 127


def _plain_values(code, biased):
    M, K = code.shape
    table = torch.tensor(_LEVELS + tuple(-v for v in _LEVELS), device=code.device)
    v = table[code.long()].view(M, K // 32, 32)
    return _times_power(v, biased.unsqueeze(2) - 127).view(M, K)


def _pack(code):
    return (code[:, 0::2] + 16 * code[:, 1::2]).to(torch.uint8)


def _unpack(q):
    q = q.int()
    return torch.stack((q % 16, q // 16), 2).view(q.shape[0], -1)


def _to_tiles(biased):
    M, blocks = biased.shape
    out = torch.zeros((blocks + 7) // 8, M, 8, device=biased.device, dtype=torch.uint8)
    for t in range(out.shape[0]):
        part = biased[:, 8 * t:8 * t + 8]
        out[t, :, :part.shape[1]] = part.to(torch.uint8)
    return out


def _from_tiles(scales, K):
    return scales.permute(1, 0, 2).reshape(scales.shape[1], -1)[:, :K // 32].int()


def _plain_held(q, scales):
    code = _unpack(q)
    return _plain_values(code, _from_tiles(scales, code.shape[1]))


# ---------------------------------------------------------------------------- cases


def prepare(case, seed):
    """Activations ~ N(0, 1), for MXFP4 with columns of their own size; weights ~ N(0, 1) / sqrt(K); gradients ~ 0.1 N(0, 1).
    Weights held in MXFP4, and what the forward pass kept for the backward pass, are in hand before the call."""
    dtype = _DTYPES[case["dtype"]]
    gen = torch.Generator(device="cuda").manual_seed(seed)
    op, M, K = case["op"], case["M"], case["K"]
    N = case.get("N", 0)

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device="cuda", dtype=dtype)

    def empty(*shape, dtype=dtype):
        return torch.empty(*shape, device="cuda", dtype=dtype)

    s = {"op": op, "a": normal(M, K)}
    if op in ("gated", "gated_bw"):
        s["b"] = normal(2 * N, K) * K ** -0.5
        if op == "gated":
            s["h"], s["gu"] = empty(M, N), empty(M, 2 * N) if case["train"] else None
        else:
            s["gu"] = (s["a"].float() @ s["b"].float().t()).to(dtype)
            s["dh"] = 0.1 * normal(M, N)
            s["da"], s["db"] = empty(M, K), empty(2 * N, K)
        return s
    s["a"] *= torch.exp(normal(K).float()).to(dtype)
    if op == "quant":
        s["q"], s["scales"] = empty(M, K // 2, dtype=torch.uint8), empty((K + 255) // 256, M, 8, dtype=torch.uint8)
        s["x"] = empty(M, K)
        return s
    code, biased = _plain_quant(normal(N, K) * K ** -0.5)
    s["b"], s["b_scales"] = _pack(code), _to_tiles(biased)
    if op == "product":
        code, biased = _plain_quant(s["a"])
        s["a"], s["a_scales"] = _pack(code), _to_tiles(biased)
    s["c"] = empty(M, N)
    return s


def _run_own(s):
    package = os.path.join(os.getcwd(), "general-nvgpu-testing_amd")
    if package not in sys.path:
        sys.path.insert(0, package)
    import beam

    op = s["op"]
    if op == "gated":
        beam.gemmrc_gated(s["a"], s["b"], s["h"], s["gu"])
        return (s["h"],) if s["gu"] is None else (s["h"], s["gu"])
    if op == "gated_bw":
        beam.gemmrc_gated_backward(s["dh"], s["gu"], s["a"], s["b"], s["da"], s["db"])
        return s["da"], s["db"]
    if op == "quant":
        beam.mxfp4_quantize(s["a"], s["q"], s["scales"])
        beam.mxfp4_dequantize(s["q"], s["scales"], s["x"])
        return s["x"], s["scales"]
    if op == "product":
        beam.gemmrc_mxfp4(s["a"], s["a_scales"], s["b"], s["b_scales"], s["c"])
    else:
        beam.linear_mxfp4(s["a"], s["b"], s["b_scales"], s["c"])
    return (s["c"],)


def run(s):
    if own:
        return _run_own(s)
    op = s["op"]
    if op == "gated":
        h, gu = _plain_gated(s["a"], s["b"])
        dtype = s["h"].dtype
        return (h.to(dtype),) if s["gu"] is None else (h.to(dtype), gu.to(dtype))
    if op == "gated_bw":
        da, db = _plain_gated_bw(s["dh"], s["gu"], s["a"], s["b"])
        return da.to(s["a"].dtype), db.to(s["b"].dtype)
    if op == "quant":
        code, biased = _plain_quant(s["a"])
        return _plain_values(code, biased).to(s["a"].dtype), _to_tiles(biased)
    a = _plain_held(s["a"], s["a_scales"]) if op == "product" else _plain_values(*_plain_quant(s["a"]))
    return ((a @ _plain_held(s["b"], s["b_scales"]).t()).to(s["c"].dtype),)


def work(case):
    op, M, K = case["op"], case["M"], case["K"]
    N = case.get("N", 0)

    def held(rows):  # bytes of a matrix of K columns in MXFP4
        return rows * (K // 2 + K // 32)

    if op == "gated":
        outputs = M * N * (3 if case["train"] else 1)
        return {"bytes": 2 * (M * K + 2 * N * K + outputs), "flops": 4 * M * N * K}
    if op == "gated_bw":
        return {"bytes": 2 * (3 * M * N + 2 * M * K + 4 * N * K), "flops": 8 * M * N * K}
    if op == "quant":
        return {"bytes": 4 * M * K + M * K // 32, "flops": 2 * M * K}
    first = held(M) if op == "product" else 2 * M * K
    return {"bytes": first + held(N) + 2 * M * N, "flops": 2 * M * N * K}


# ---------------------------------------------------------------------------- the definitions, in 64 bits


def _exact_power(e):
    table = torch.tensor([2.0 ** n for n in range(-160, 161)], device=e.device, dtype=torch.float64)
    return table[e.long() + 160]


def _exact_mx(x):
    """Values [M, K] that MXFP4 holds for x, and the biased exponents [M, K / 32]: the block's power of two is that of its
    largest magnitude over 4, an element is the magnitude nearest to it, the one with an even code of two as near."""
    M, K = x.shape
    v = x.double().view(M, K // 32, 32)
    top = v.abs().amax(2, keepdim=True)
    e = torch.floor(torch.log2(top))
    e = torch.where(top > 0, e, torch.full_like(e, -125.0))
    e = torch.where(_exact_power(e) > top, e - 1, e)
    e = torch.where(_exact_power(e + 1) <= top, e + 1, e) - 2
    e = torch.where(top > 0, e, torch.full_like(e, -127.0)).clamp(min=-127.0)
    y = v.abs() * _exact_power(-e)
    best = torch.zeros_like(y)
    gap = y.clone()
    for i, level in list(enumerate(_LEVELS))[1:]:
        d = (y - level).abs()
        nearer = (d < gap) | ((d == gap) & (i % 2 == 0))
        best, gap = torch.where(nearer, torch.full_like(best, level), best), torch.where(nearer, d, gap)
    return (torch.where(v < 0, -best, best) * _exact_power(e)).view(M, K), (e.squeeze(2) + 127).int()


def _exact_held(q, scales):
    rows, K = q.shape[0], 2 * q.shape[1]
    levels = torch.tensor(_LEVELS, device=q.device, dtype=torch.float64)
    out = torch.empty(rows, K, device=q.device, dtype=torch.float64)
    for half in range(2):
        code = (q.long() >> (4 * half)) & 15
        out[:, half::2] = levels[code & 7] * (1 - 2 * (code >> 3)).double()
    for block in range(K // 32):
        out[:, 32 * block:32 * block + 32] *= _exact_power(scales[block // 8, :, block % 8].int() - 127).unsqueeze(1)
    return out


def exact(case, seed):
    s = prepare(case, seed)
    op = s["op"]
    if op in ("gated", "gated_bw"):
        a, b = s["a"].double(), s["b"].double()
        N = case["N"]
        if op == "gated":
            g, u = a @ b[:N].t(), a @ b[N:].t()
            h = u * g * torch.sigmoid(g)
            return (h, torch.cat((g, u), 1)) if case["train"] else (h,)
        g, u, dh = s["gu"][:, :N].double(), s["gu"][:, N:].double(), s["dh"].double()
        sig = torch.sigmoid(g)
        dg = dh * u * (sig + g * sig * torch.sigmoid(-g))
        du = dh * g * sig
        return dg @ b[:N] + du @ b[N:], torch.cat((dg.t() @ a, du.t() @ a), 0)
    if op == "quant":
        values, biased = _exact_mx(s["a"])
        scales = torch.zeros_like(s["scales"])
        for block in range(biased.shape[1]):
            scales[block // 8, :, block % 8] = biased[:, block].to(torch.uint8)
        return values, scales
    a = _exact_held(s["a"], s["a_scales"]) if op == "product" else _exact_mx(s["a"])[0]
    return (a @ _exact_held(s["b"], s["b_scales"]).t(),)
