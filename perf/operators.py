"""The microscaled-format operators, measured: block quantisation, reading back, the product of two
quantised matrices, and the root-mean-square norm that quantises its output.

A matrix in one of these formats is (codes, scales): every block of 32 consecutive elements of a row
shares a power of two, 2^(scale - 127), and each element is a 4-bit float (e2m1, two to a byte, the
even element in the low half) or an 8-bit one (e4m3).  Scales come row by row, (rows, K / 32), or in the
order the tensor cores read them, one 512-byte record per 128 rows x 128 columns.
"""
import math

import torch

own = False

BLOCK = 32
EMAX = {4: 2, 8: 8}            # exponent of the element type's largest power of two
LARGEST = {4: 6.0, 8: 448.0}
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}


def _s24():
    import os
    import sys
    path = os.path.join(os.getcwd(), "gpu-compression-kernel_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import s24
    return s24


def listed():
    return [
        # activations of one decoding step of a batch of 64, for a 4-bit product; read back for a unit that wants 16 bits
        {"name": "quantize4 step", "op": "quantize", "bits": 4, "rows": 64, "k": 4096, "dtype": "bf16"},
        # a whole MLP weight turned into 4 bits when a model is loaded, and read back to look at the error
        {"name": "quantize4 weight", "op": "quantize", "bits": 4, "rows": 28672, "k": 8192, "dtype": "bf16"},
        # a prompt's activations for an 8-bit product
        {"name": "quantize8 prompt", "op": "quantize", "bits": 8, "rows": 8192, "k": 8192, "dtype": "fp16"},
        # a 4-bit weight expanded for a layer that computes in 16 bits
        {"name": "dequantize4 weight", "op": "dequantize", "bits": 4, "rows": 16384, "k": 16384, "dtype": "bf16"},
        # 8-bit activations of a ragged batch read back
        {"name": "dequantize8 ragged", "op": "dequantize", "bits": 8, "rows": 1537, "k": 4128, "dtype": "fp16"},
        # the norm before a linear layer, one decoding step of 16 sequences
        {"name": "norm8 step", "op": "norm", "bits": 8, "rows": 16, "k": 8192, "dtype": "bf16", "residual": True},
        # the same for a prompt
        {"name": "norm8 prompt", "op": "norm", "bits": 8, "rows": 8192, "k": 8192, "dtype": "bf16", "residual": True},
        # the first norm of a network (no residual yet) over a ragged batch, output in 4 bits
        {"name": "norm4 ragged", "op": "norm", "bits": 4, "rows": 4099, "k": 6144, "dtype": "fp16", "residual": False},
        # the framework's headline product size, both sides in 4 bits
        {"name": "product44 square", "op": "product", "bits_a": 4, "bits_b": 4, "m": 8192, "n": 8192, "k": 8192, "dtype": "bf16"},
        # the MLP's up projection for a ragged prompt: 8-bit activations, 4-bit weight
        {"name": "product84 prompt", "op": "product", "bits_a": 8, "bits_b": 4, "m": 4001, "n": 28672, "k": 8192, "dtype": "bf16"},
        # the same weight in a decoding step of four sequences: reading the weight is the work
        {"name": "product84 step", "op": "product", "bits_a": 8, "bits_b": 4, "m": 4, "n": 28672, "k": 8192, "dtype": "bf16"},
        # both sides in 8 bits, nothing a multiple of a tile
        {"name": "product88 ragged", "op": "product", "bits_a": 8, "bits_b": 8, "m": 1537, "n": 6150, "k": 4128, "dtype": "fp16"},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(("quantize", "dequantize", "norm", "product", "product"))
    dtype = rng.choice(("bf16", "fp16"))
    if op == "product":
        bits_a, bits_b = rng.choice(((4, 4), (8, 4), (8, 8)))
        step = 128 if bits_a != bits_b else 32
        while True:
            case = {"op": op, "bits_a": bits_a, "bits_b": bits_b, "m": _log(rng, 1, 8192), "n": _log(rng, 64, 28672),
                    "k": step * max(1, _log(rng, 128, 16384) // step), "dtype": dtype}
            if case["m"] * case["n"] * case["k"] <= 8192 ** 3:
                return case
    bits = rng.choice((4, 8))
    if op == "norm":
        while True:
            case = {"op": op, "bits": bits, "rows": _log(rng, 1, 16384), "k": 32 * max(1, _log(rng, 128, 16384) // 32),
                    "dtype": dtype, "residual": rng.random() < 0.7}
            if case["rows"] * case["k"] <= 8192 * 8192:
                return case
    if op == "quantize":
        dtype = rng.choice(("bf16", "fp16", "fp32"))
    while True:
        case = {"op": op, "bits": bits, "rows": _log(rng, 1, 28672), "k": 32 * max(1, _log(rng, 32, 16384) // 32), "dtype": dtype}
        if case["rows"] * case["k"] <= 8192 * 8192:
            return case


# ------------------------------------------------------------------ plain form

def _round_to(v, bits):
    """v rounded to the element type, half to even, saturating; in v's own precision"""
    mag = v.abs()
    low, fraction = (0, 1) if bits == 4 else (-6, 3)
    e = (torch.frexp(mag)[1] - 1).clamp(min=low)
    step = torch.ldexp(torch.ones_like(v), e - fraction)
    return torch.copysign((torch.round(mag / step) * step).clamp(max=LARGEST[bits]), v)


def _quantize(x, bits):
    """element values (rows, K) and biased scale exponents (rows, K / 32) of x, in x's precision"""
    blocks = x.reshape(x.shape[0], -1, BLOCK)
    amax = blocks.abs().amax(-1)
    code = (torch.frexp(amax)[1] - 1 - EMAX[bits] + 127).clamp(0, 254)
    code = torch.where(amax == 0, torch.zeros_like(code), code)
    up = torch.ldexp(torch.ones_like(amax), 127 - code)
    ok = torch.isfinite(amax)
    q = _round_to(blocks * up.unsqueeze(-1), bits)
    q = torch.where(ok.unsqueeze(-1), q, torch.zeros_like(q))
    return q.reshape(x.shape), torch.where(ok, code, torch.full_like(code, 255)).to(torch.uint8)


def _scale_value(scales):
    """2^(scale - 127), NaN for 255"""
    v = torch.ldexp(torch.ones_like(scales, dtype=torch.float32), scales.to(torch.int32) - 127)
    return torch.where(scales == 255, torch.full_like(v, math.nan), v)


def _tensor_core_order(scales):
    """(rows, K / 32) scales as the records the product reads; positions outside the matrix are 0"""
    r, kb = scales.shape
    tiles, chunks = -(-r // 128), -(-kb // 4)
    full = torch.zeros((tiles * 128, chunks * 4), dtype=scales.dtype, device=scales.device)
    full[:r, :kb] = scales
    return full.view(tiles, 4, 32, chunks, 4).permute(0, 3, 2, 1, 4).contiguous().view(-1)


def _pack(q):
    """4-bit element values as bytes, the even element in the low half"""
    mag = q.abs()
    code = torch.where(mag < 2, mag * 2, torch.where(mag < 4, mag + 2, mag * 0.5 + 4)).to(torch.uint8)
    code = code | (torch.signbit(q).to(torch.uint8) << 3)
    return code[:, 0::2] | (code[:, 1::2] << 4)


def _elements(codes):
    """element values of codes in 32 bits"""
    if codes.dtype == torch.float8_e4m3fn:
        return codes.to(torch.float32)
    both = torch.stack((codes & 15, codes >> 4), -1).reshape(codes.shape[0], -1)
    mag = (both & 7).to(torch.float32)
    mag = torch.where(mag < 4, mag * 0.5, torch.where(mag < 6, mag - 2, mag * 2 - 8))
    return torch.where(both > 7, -mag, mag)


def _read_back(codes, scales):
    v = _elements(codes)
    return (v.view(v.shape[0], -1, BLOCK) * _scale_value(scales).unsqueeze(-1)).view(v.shape)


# ------------------------------------------------------------------ the calls that are measured

def _activations(rows, k, g, device):
    """what leaves a residual stream: a few channels much larger than the others, some padded rows"""
    x = torch.randn(rows, k, generator=g, device=device)
    channel = torch.exp(0.5 * torch.randn(k, generator=g, device=device))
    channel[torch.rand(k, generator=g, device=device) < 0.005] *= 20.0
    x *= channel
    if rows > 32:
        x[torch.rand(rows, generator=g, device=device) < 0.01] = 0.0
    return x


def _operand(rows, k, bits, activations, g, device):
    x = _activations(rows, k, g, device) if activations else 0.02 * torch.randn(rows, k, generator=g, device=device)
    q, scales = _quantize(x, bits)
    codes = _pack(q) if bits == 4 else q.to(torch.float8_e4m3fn)
    return {"codes": codes, "scales": scales, "scales_tc": _tensor_core_order(scales)}


def prepare(case, seed):
    device = torch.device("cuda")
    g = torch.Generator(device=device).manual_seed(seed)
    op, dtype = case["op"], DTYPES[case["dtype"]]
    state = {"case": dict(case)}
    if op == "product":
        state["a"] = _operand(case["m"], case["k"], case["bits_a"], True, g, device)
        state["b"] = _operand(case["n"], case["k"], case["bits_b"], False, g, device)
    elif op == "dequantize":
        state["x"] = _operand(case["rows"], case["k"], case["bits"], case["rows"] < 8192, g, device)
    else:
        state["x"] = _activations(case["rows"], case["k"], g, device).to(dtype)
        if op == "norm":
            state["weight"] = (1.0 + 0.1 * torch.randn(case["k"], generator=g, device=device)).to(dtype)
            state["residual"] = _activations(case["rows"], case["k"], g, device).to(dtype) if case["residual"] else None
    return state


EPS = 1e-6


def run(state):
    case = state["case"]
    op, dtype = case["op"], DTYPES[case["dtype"]]
    if own:
        s24 = _s24()
        if op == "product":
            a, b = state["a"], state["b"]
            return s24.mx_matmul(a["codes"], a["scales_tc"], b["codes"], b["scales_tc"], out_dtype=dtype)
        if op == "dequantize":
            return s24.mx_dequantize(state["x"]["codes"], state["x"]["scales"], dtype=dtype)
        fmt = "mxfp4" if case["bits"] == 4 else "mxfp8"
        if op == "quantize":
            codes, _, tc = s24.mx_quantize(state["x"], fmt, want_rows=False, want_tc=True)
            if case["bits"] == 4:
                return s24.mx_dequantize(codes, tc, layout="tc", dtype=torch.float32 if dtype == torch.float32 else torch.bfloat16)
            return codes, tc.view(torch.float8_e8m0fnu)
        codes, scales, _, h = s24.mx_rms_norm(state["x"], state["weight"], eps=EPS, residual=state["residual"], fmt=fmt)
        if case["bits"] == 4:
            return h, s24.mx_dequantize(codes, scales, dtype=torch.bfloat16)
        return h, codes, scales.view(torch.float8_e8m0fnu)
    if op == "product":
        a, b = (_read_back(x["codes"], x["scales"]) for x in (state["a"], state["b"]))
        return (a @ b.t()).to(dtype)
    if op == "dequantize":
        return _read_back(state["x"]["codes"], state["x"]["scales"]).to(dtype)
    if op == "quantize":
        q, scales = _quantize(state["x"].float(), case["bits"])
        if case["bits"] == 4:
            return _read_back(_pack(q), scales).to(torch.float32 if dtype == torch.float32 else torch.bfloat16)
        return q.to(torch.float8_e4m3fn), _tensor_core_order(scales).view(torch.float8_e8m0fnu)
    # the norm: what is rounded to 8 or 4 bits lies next to a border for some element of any large input, so 64 bits
    h = state["x"]
    if state["residual"] is not None:
        h = (h.float() + state["residual"].float()).to(dtype)
    wide = h.double()
    y = wide * torch.rsqrt(wide.square().mean(-1, keepdim=True) + EPS) * state["weight"].double()
    q, scales = _quantize(y, case["bits"])
    if case["bits"] == 4:
        return h, _read_back(_pack(q), scales).to(torch.bfloat16)
    return h, q.to(torch.float8_e4m3fn), scales.view(torch.float8_e8m0fnu)


def work(case):
    op = case["op"]
    if op == "product":
        m, n, k = case["m"], case["n"], case["k"]
        operand = m * k * (case["bits_a"] / 8 + 1 / BLOCK) + n * k * (case["bits_b"] / 8 + 1 / BLOCK)
        return {"bytes": operand + m * n * SIZE[case["dtype"]], "flops": 2.0 * m * n * k}
    n = case["rows"] * case["k"]
    packed, wide = n * (case["bits"] / 8 + 1 / BLOCK), n * SIZE[case["dtype"]]
    if op == "dequantize":
        return {"bytes": packed + wide, "flops": float(n)}
    read_back = packed + n * (4 if case["dtype"] == "fp32" else 2) if case["bits"] == 4 else 0
    if op == "quantize":
        return {"bytes": wide + packed + read_back, "flops": 3.0 * n}
    # x, the residual and the new residual; without a residual h is x itself
    return {"bytes": wide * (3 if case["residual"] else 1) + packed + read_back + case["k"] * SIZE[case["dtype"]], "flops": 7.0 * n}


# ------------------------------------------------------------------ the definition in 64 bits

def _table(bits, device):
    """the element type's values from 0 upwards; a value's place in the table has its last bit of fraction"""
    fraction, low, top = (1, 0, 2) if bits == 4 else (3, -6, 8)
    n = 1 << fraction
    values = [2.0 ** low * i / n for i in range(n)] + [2.0 ** e * (1 + i / n) for e in range(low, top + 1) for i in range(n)]
    return torch.tensor([v for v in values if v <= LARGEST[bits]], dtype=torch.float64, device=device)


def _exact_quantize(v, bits):
    """(element values, powers of two of the blocks) of v, 64 bits"""
    device = v.device
    t = _table(bits, device)
    middle = (t[1:] + t[:-1]) / 2
    powers = torch.tensor([2.0 ** e for e in range(-126 + EMAX[bits], 129)], dtype=torch.float64, device=device)
    blocks = v.reshape(v.shape[0], -1, BLOCK)
    place = torch.searchsorted(powers, blocks.abs().amax(-1).contiguous(), right=True)   # 0: below 2^(emax - 126)
    scale = torch.tensor([2.0 ** e for e in range(-127, 128)], dtype=torch.float64, device=device)[place]
    mag = (blocks / scale.unsqueeze(-1)).abs()
    low, high = torch.searchsorted(middle, mag), torch.searchsorted(middle, mag, right=True)
    q = t[torch.where((low != high) & (low % 2 == 1), high, low)] * torch.sign(blocks)
    return q.view(v.shape), scale


def _exact_values(codes, scales):
    if codes.dtype == torch.float8_e4m3fn:
        t = _table(8, codes.device)
        t = torch.cat((t, torch.full((1,), math.nan, dtype=torch.float64, device=codes.device)))
        c, sign = codes.view(torch.uint8), 128
    else:
        t = _table(4, codes.device)
        c, sign = torch.empty((codes.shape[0], 2 * codes.shape[1]), dtype=torch.uint8, device=codes.device), 8
        c[:, 0::2], c[:, 1::2] = codes % 16, codes // 16
    v = t[(c % sign).long()] * torch.where(c < sign, 1.0, -1.0).double()
    s = torch.tensor([2.0 ** (e - 127) for e in range(255)] + [math.nan], dtype=torch.float64, device=codes.device)[scales.long()]
    return (v.view(v.shape[0], -1, BLOCK) * s.unsqueeze(-1)).view(v.shape)


def _exact_tensor_core_order(scale):
    """as records, by each position's own place"""
    r, kb = scale.shape
    chunks = -(-kb // 4)
    i = torch.arange(r, device=scale.device).unsqueeze(1)
    j = torch.arange(kb, device=scale.device).unsqueeze(0)
    at = ((i // 128) * chunks + j // 4) * 512 + (i % 32) * 16 + (i % 128) // 32 * 4 + j % 4
    out = torch.full((-(-r // 128) * chunks * 512,), 2.0 ** -127, dtype=torch.float64, device=scale.device)
    out[at] = scale
    return out


def exact(case, seed):
    state = prepare(case, seed)
    op = case["op"]
    if op == "product":
        a, b = (_exact_values(state[x]["codes"], state[x]["scales"]) for x in ("a", "b"))
        return a @ b.t()
    if op == "dequantize":
        return _exact_values(state["x"]["codes"], state["x"]["scales"])
    if op == "quantize":
        q, scale = _exact_quantize(state["x"].double(), case["bits"])
        if case["bits"] == 4:
            return (q.view(q.shape[0], -1, BLOCK) * scale.unsqueeze(-1)).view(q.shape)
        return q, _exact_tensor_core_order(scale)
    h = state["x"].double()
    if state["residual"] is not None:
        h = (h + state["residual"].double()).to(DTYPES[case["dtype"]]).double()
    y = h / torch.sqrt((h * h).sum(-1, keepdim=True) / h.shape[1] + EPS) * state["weight"].double()
    q, scale = _exact_quantize(y, case["bits"])
    if case["bits"] == 4:
        return h, (q.view(q.shape[0], -1, BLOCK) * scale.unsqueeze(-1)).view(q.shape)
    return h, q, scale
