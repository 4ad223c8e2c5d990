"""Cases, plain forms and 64-bit definitions of the block-scaled (MX) operators.

A transformer layer that keeps its weights in 4 bits and the activations
between its kernels in 8 bits runs four operators:

``norm``   the residual's addition, RMSNorm, and an output in 8 bits with scales
``quant``  an activation written in 8 bits with scales (what attention returns)
``gemm``   a product with 4-bit weights: out = a @ dequant(b)^T
``gated``  act(a @ gate^T) * (a @ up^T) with 4-bit weights, in 16 or 8 bits

Both formats share one scale, a power of two held as its biased exponent in a
byte, among 32 neighbours of a row:

    8 bits: e4m3 values, scale 2^e with the least e for which max|x| <= 448 * 2^e
    4 bits: e2m1 values (0, .5, 1, 1.5, 2, 3, 4, 6), two in a byte, even k low

A block that holds a NaN or an infinity is NaN throughout (scale byte 255).
"""
import math

import torch

own = False

BLOCK = 32
_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
_framework = None


def _fi():
    global _framework
    if _framework is None:
        import flashinfer_amd

        _framework = flashinfer_amd
    return _framework


def listed():
    return [
        # one request, one new token: the norm in front of every projection
        {"name": "norm_token", "op": "norm", "m": 1, "k": 4096, "dtype": "bf16", "add": True},
        # a decode batch of odd size without a residual (the first layer, or a q/k latent norm)
        {"name": "norm_batch_odd", "op": "norm", "m": 251, "k": 7168, "dtype": "fp16", "add": False},
        # a long prefill through a wide model
        {"name": "norm_prefill", "op": "norm", "m": 16384, "k": 8192, "dtype": "bf16", "add": True},
        # what attention returns for a decode batch, ahead of the output projection
        {"name": "quant_batch", "op": "quant", "m": 64, "k": 4096, "dtype": "bf16"},
        # the same for a chunk of prefill, with a row count that no tile divides
        {"name": "quant_prefill_odd", "op": "quant", "m": 8191, "k": 14336, "dtype": "fp16"},
        # the fused q/k/v projection of a single token
        {"name": "gemm_token", "op": "gemm", "m": 1, "n": 6144, "k": 4096, "dtype": "bf16", "act8": False},
        # the down projection of a decode batch, fed in 8 bits by the gated block
        {"name": "gemm_batch_act8", "op": "gemm", "m": 16, "n": 4096, "k": 14336, "dtype": "bf16", "act8": True},
        # a vocabulary of odd size at a few rows (the head of a small batch)
        {"name": "gemm_head_odd", "op": "gemm", "m": 5, "n": 32001, "k": 4096, "dtype": "fp16", "act8": False},
        # the down projection of a prefill chunk, in 8 bits
        {"name": "gemm_prefill_act8", "op": "gemm", "m": 4096, "n": 4096, "k": 14336, "dtype": "bf16", "act8": True},
        # the feed-forward block's first half for a single token
        {"name": "gated_token", "op": "gated", "m": 1, "n": 14336, "k": 4096, "dtype": "bf16", "act8": False, "act": "silu", "out8": False},
        # the same for a decode batch, 8 bits in and 8 bits out
        {"name": "gated_batch_act8", "op": "gated", "m": 48, "n": 14336, "k": 4096, "dtype": "bf16", "act8": True, "act": "silu", "out8": True},
        # a ragged prefill chunk with 16-bit activations
        {"name": "gated_prefill_odd", "op": "gated", "m": 2047, "n": 14336, "k": 4096, "dtype": "bf16", "act8": False, "act": "gelu_tanh", "out8": False},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["norm", "quant", "gemm", "gemm", "gated", "gated"])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    if op in ("norm", "quant"):
        k = BLOCK * _log(rng, 8, 448)
        m = _log(rng, 1, min(16384, (16384 * 8192) // k))
        case = {"op": op, "m": m, "k": k, "dtype": dtype}
        if op == "norm":
            case["add"] = rng.random() < 0.7
        return case
    k = BLOCK * _log(rng, 8, 448)
    m = _log(rng, 1, 4096)
    # no more multiplications than the largest listed product
    most = 4096 * 4096 * 14336 // (m * k)
    n = _log(rng, 64, max(64, min(32768, most) // (2 if op == "gated" else 1)))
    case = {"op": op, "m": m, "n": n, "k": k, "dtype": dtype, "act8": rng.random() < 0.5}
    if op == "gated":
        case["act"] = rng.choice(["silu", "silu", "gelu", "gelu_tanh"])
        case["out8"] = rng.random() < 0.5
        if case["out8"]:
            case["n"] = max(BLOCK, n // BLOCK * BLOCK)
    return case


# ---------------------------------------------------------------- inputs

def _hidden(gen, m, k, size):
    """Activations: normal values, channels of unlike size, a few of them large."""
    dev = "cuda"
    channel = torch.exp(0.3 * torch.randn(k, generator=gen, device=dev))
    channel[torch.rand(k, generator=gen, device=dev) < 0.002] *= 20.0
    return torch.randn(m, k, generator=gen, device=dev) * (channel * size)


def _weight4(gen, n, k):
    """Weights of a trained projection, in 4 bits: rows of unlike size, two
    values in a byte, and the scales' exponents."""
    dev = "cuda"
    packed = torch.empty(n, k // 2, dtype=torch.uint8, device=dev)
    scale = torch.empty(n, k // BLOCK, dtype=torch.uint8, device=dev)
    step = max(1, (1 << 27) // k)
    for at in range(0, n, step):
        rows = min(step, n - at)
        row = torch.exp(0.3 * torch.randn(rows, 1, generator=gen, device=dev)) / math.sqrt(k)
        w = (torch.randn(rows, k, generator=gen, device=dev) * row).view(rows, k // BLOCK, BLOCK)
        mantissa, exponent = torch.frexp(w.abs().amax(-1))
        # frexp's mantissa is in [.5, 1): 6 = .75 * 2^3
        exponent = exponent - 3 + (mantissa > 0.75)
        exponent = exponent.clamp(-127, 127)
        scaled = torch.ldexp(w, -exponent.unsqueeze(-1))
        edges = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], device=dev)
        code = torch.bucketize(scaled.abs(), edges).to(torch.uint8) | ((scaled < 0).to(torch.uint8) << 3)
        code = code.view(rows, k)
        packed[at:at + rows] = code[:, 0::2] | (code[:, 1::2] << 4)
        scale[at:at + rows] = (exponent + 127).to(torch.uint8)
    return packed, scale


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    dtype, m, k = _DTYPES[case["dtype"]], case["m"], case["k"]
    state = dict(case)
    if case["op"] == "norm":
        # what a layer adds to the residual is smaller than the residual
        state["x"] = _hidden(gen, m, k, 0.1 if case["add"] else 1.0).to(dtype)
        if case["add"]:
            state["residual"] = _hidden(gen, m, k, 1.0).to(dtype)
        state["weight"] = (1.0 + 0.2 * torch.randn(k, generator=gen, device="cuda")).to(dtype)
        return state
    x = _hidden(gen, m, k, 1.0)
    if case["op"] == "quant":
        state["x"] = x.to(dtype)
        return state
    if case["act8"]:
        state["x"], state["x_scale"] = _to8(x)
    else:
        state["x"] = x.to(dtype)
    rows = 2 * case["n"] if case["op"] == "gated" else case["n"]
    state["w"], state["w_scale"] = _weight4(gen, rows, k)
    return state


# ---------------------------------------------------------------- plain forms

def _to8(y):
    """y (32-bit) as e4m3 values and exponent bytes, one for 32 neighbours."""
    blocks = y.view(y.shape[0], -1, BLOCK)
    most = blocks.abs().amax(-1)
    mantissa, exponent = torch.frexp(most)
    # frexp's mantissa is in [.5, 1): 448 = .875 * 2^9
    exponent = (exponent - 9 + (mantissa > 0.875)).clamp(min=-127)
    exponent = torch.where(most == 0, torch.full_like(exponent, -127), exponent)
    bad = ~torch.isfinite(most)
    exponent = torch.where(bad, torch.zeros_like(exponent), exponent)
    q = torch.ldexp(blocks, -exponent.unsqueeze(-1))
    q = torch.where(bad.unsqueeze(-1), torch.full_like(q, math.nan), q)
    scale = torch.where(bad, torch.full_like(exponent, 128), exponent) + 127
    return q.view_as(y).to(torch.float8_e4m3fn), scale.to(torch.uint8)


def _exponent_value(byte):
    """2^(byte - 127) in 32 bits; 255 is NaN."""
    bits = byte.to(torch.int32) << 23
    bits = torch.where(byte == 0, torch.full_like(bits, 0x00400000), bits)
    bits = torch.where(byte == 255, torch.full_like(bits, 0x7FC00000), bits)
    return bits.view(torch.float32)


def _from8(q, scale):
    s = _exponent_value(scale).unsqueeze(-1)
    return (q.float().view(q.shape[0], -1, BLOCK) * s).view(q.shape)


def _from4(packed, scale):
    levels = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6, -0.0, -.5, -1, -1.5, -2, -3, -4, -6], device=packed.device)
    n, k = packed.shape[0], packed.shape[1] * 2
    code = torch.stack((packed & 15, packed >> 4), -1).view(n, k)
    w = levels[code.int()].view(n, -1, BLOCK)
    return (w * _exponent_value(scale).unsqueeze(-1)).view(n, k)


def _activate(g, act):
    if act == "silu":
        return g / (1.0 + torch.exp(-g))
    if act == "gelu":
        return 0.5 * g * (1.0 + torch.erf(g * math.sqrt(0.5)))
    return 0.5 * g * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (g + 0.044715 * g * g * g)))


def _plain(s):
    dtype = _DTYPES[s["dtype"]]
    if s["op"] == "norm":
        x = s["x"]
        if s["add"]:
            s["residual"].copy_((x.float() + s["residual"].float()).to(dtype))
            x = s["residual"]
        xf = x.float()
        y = xf * torch.rsqrt((xf * xf).mean(-1, keepdim=True) + 1e-6) * s["weight"].float()
        q, scale = _to8(y)
        return (q, scale.view(torch.float8_e8m0fnu)) + ((s["residual"],) if s["add"] else ())
    if s["op"] == "quant":
        q, scale = _to8(s["x"].float())
        return q, scale.view(torch.float8_e8m0fnu)
    a = _from8(s["x"], s["x_scale"]) if s["act8"] else s["x"].float()
    w = _from4(s["w"], s["w_scale"])
    if s["op"] == "gemm":
        return (a @ w.t()).to(dtype)
    n = s["n"]
    y = _activate(a @ w[:n].t(), s["act"]) * (a @ w[n:].t())
    if not s["out8"]:
        return y.to(dtype)
    q, scale = _to8(y)
    return q, scale.view(torch.float8_e8m0fnu)


def run(state):
    if not own:
        return _plain(state)
    fi, s = _fi(), state
    if s["op"] == "norm":
        if s["add"]:
            q, scale = fi.fused_add_rmsnorm_mxfp8_quant(s["x"], s["residual"], s["weight"])
            return q, scale.view(torch.float8_e8m0fnu), s["residual"]
        q, scale = fi.rmsnorm_mxfp8_quant(s["x"], s["weight"])
        return q, scale.view(torch.float8_e8m0fnu)
    if s["op"] == "quant":
        q, scale = fi.mxfp8_quantize(s["x"])
        return q, scale.view(torch.float8_e8m0fnu)
    dtype = _DTYPES[s["dtype"]]
    if s["op"] == "gemm":
        return fi.gemm_mxfp4_nt(s["x"], s["w"], s["w_scale"], s.get("x_scale"), out_dtype=dtype)
    if not s["out8"]:
        return fi.gemm_mxfp4_nt_gated(s["x"], s["w"], s["w_scale"], s.get("x_scale"), activation=s["act"], out_dtype=dtype)
    q, scale = fi.gemm_mxfp4_nt_gated(s["x"], s["w"], s["w_scale"], s.get("x_scale"), activation=s["act"], out_dtype=torch.float8_e4m3fn)
    return q, scale.view(torch.float8_e8m0fnu)


# ---------------------------------------------------------------- definitions in 64 bits

def _power(byte):
    """2^(byte - 127) in 64 bits, from the bits of a double."""
    value = ((byte.to(torch.int64) - 127 + 1023) << 52).view(torch.float64)
    return torch.where(byte == 255, torch.full_like(value, math.nan), value)


def _exact8(y):
    """The unrounded values in units of their scale, and the scale, both in 64 bits."""
    blocks = y.reshape(y.shape[0], -1, BLOCK)
    most = blocks.abs().amax(-1)
    e = torch.ceil(torch.log2(most / 448.0))
    # the logarithm may be off by an ulp next to a whole number
    e = torch.where(448.0 * torch.exp2(e - 1) >= most, e - 1, e)
    e = torch.where(448.0 * torch.exp2(e) < most, e + 1, e)
    e = torch.where(most == 0, torch.full_like(e, -127.0), e.clamp(min=-127.0))
    s = torch.exp2(e)
    return (blocks / s.unsqueeze(-1)).reshape(y.shape), s


def _exact_rows4(packed, scale):
    """e2m1 by its definition: sign, two bits of exponent with bias 1, one of mantissa."""
    n = packed.shape[0]
    code = torch.empty(n, packed.shape[1], 2, dtype=torch.int64, device=packed.device)
    code[..., 0] = packed % 16
    code[..., 1] = packed // 16
    sign = 1.0 - 2.0 * (code // 8).double()
    exponent, mantissa = (code // 2) % 4, (code % 2).double()
    normal = (1.0 + mantissa / 2.0) * torch.exp2(exponent.double() - 1.0)
    value = sign * torch.where(exponent == 0, mantissa / 2.0, normal)
    return value.reshape(n, -1) * _power(scale).repeat_interleave(BLOCK, dim=1)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "norm":
        x, done = s["x"].double(), ()
        if case["add"]:
            total = x + s["residual"].double()
            done = (total,)
            x = total.to(_DTYPES[case["dtype"]]).double()  # the residual is held in its own type
        root = torch.sqrt(x.square().sum(-1, keepdim=True) / case["k"] + 1e-6)
        return _exact8(x / root * s["weight"].double()) + done
    if case["op"] == "quant":
        return _exact8(s["x"].double())
    a = s["x"].double()
    if case["act8"]:
        a = a * _power(s["x_scale"]).repeat_interleave(BLOCK, dim=1)
    n, step = case["n"], 2048
    parts = []
    for at in range(0, n, step):
        to = min(n, at + step)
        part = a @ _exact_rows4(s["w"][at:to], s["w_scale"][at:to]).T
        if case["op"] == "gated":
            up = a @ _exact_rows4(s["w"][n + at:n + to], s["w_scale"][n + at:n + to]).T
            if case["act"] == "silu":
                part = part * torch.sigmoid(part)
            elif case["act"] == "gelu":
                part = part * torch.special.ndtr(part)
            else:
                part = part * torch.sigmoid(2.0 * math.sqrt(2.0 / math.pi) * (part + 0.044715 * part ** 3))
            part = part * up
        parts.append(part)
    y = torch.cat(parts, dim=1)
    return _exact8(y) if case.get("out8") else y


# ---------------------------------------------------------------- what a pass cannot do without

def work(case):
    m, k = case["m"], case["k"]
    eight = 1 + 1 / BLOCK
    four = 0.5 + 1 / BLOCK
    if case["op"] == "norm":
        moved = m * k * (2 * (3 if case["add"] else 1) + eight) + 2 * k
        return {"bytes": moved, "flops": m * k * (6 if case["add"] else 5)}
    if case["op"] == "quant":
        return {"bytes": m * k * (2 + eight), "flops": 2 * m * k}
    n, rows = case["n"], case["n"] * (2 if case["op"] == "gated" else 1)
    moved = m * k * (eight if case["act8"] else 2) + rows * k * four + m * n * (eight if case.get("out8") else 2)
    return {"bytes": moved, "flops": 2 * m * rows * k}
