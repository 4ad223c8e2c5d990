"""What the MXFP4 products add up, on operands whose sums are exact in 32 bits.

In every 128 of K one large value meets 6 and -6 in neighbouring places: the two
products cancel. The others are whole halves. A sum in units of a half stays below
2^23 of them, so 32 bits hold every partial sum in any order without a rounding,
and the result is the definition's, rounded once: to the output's type, or (gated)
to 32 bits by the product of both halves, and then to MXFP8. A sum that keeps less
below its largest product loses the small ones."""
import pytest
import torch

from test_mx import FP8, BLOCK, from4, from8, gpu, to8_bits

KINDS = {"bf16": torch.bfloat16, "fp16": torch.float16}


def exact_tokens(m, k, kind, gen):
    """(a, a_scale or None, values in 64 bits): 1, 2 or 3, and two large ones in 128."""
    v = torch.randint(1, 4, (m, k), device="cuda", generator=gen).double()
    big = 448.0 * 2 ** (6 if kind == "fp16" else 9)
    at = torch.arange(0, k, 128, device="cuda")
    at = at + at // 128 % 16 * 2  # another place of each 128, the pair within eight
    at = at[at + 1 < k]
    v[:, at] = big
    v[:, at + 1] = big
    if kind != "fp8":
        return v.to(KINDS[kind]), None, v, at
    # 448 * 2^9 beside 1: 2^-9 of the scale, the least value of e4m3
    s = torch.where(v.unflatten(1, (-1, BLOCK)).amax(-1) > 448, 136, 127).to(torch.uint8)
    q = torch.ldexp(v, 127 - s.long().repeat_interleave(BLOCK, 1)).float().to(FP8)
    assert torch.equal(from8(q, s), v)
    return q, s, v, at


def exact_weights(n, k, at, gen, positive):
    """(b, b_scale, values in 64 bits): any levels beside 6, -6 for the large tokens."""
    code = torch.randint(0, 16, (n, k), device="cuda", generator=gen)
    if positive:
        code[:n // 2] &= 7  # the gate rows
    code[:, at] = 7
    code[:, at + 1] = 15
    b = (code[:, 0::2] | code[:, 1::2] << 4).to(torch.uint8)
    b_scale = torch.full((n, k // BLOCK), 127, dtype=torch.uint8, device="cuda")
    return b, b_scale, from4(b, b_scale)


# one token to thousands: the kernel for few tokens and every tile, whole and in
# parts of K, and a K that 128 does not divide
OUT8 = [(1, 64, 4096), (7, 7008, 160), (12, 96, 6176), (16, 64, 4096), (20, 2048, 1056), (32, 9632, 128),
        (33, 64, 4096), (48, 1408, 1056), (64, 2080, 96), (100, 4256, 96), (128, 320, 6176),
        (129, 96, 4128), (129, 4256, 96), (200, 1568, 288), (200, 8480, 96), (260, 320, 6176),
        (390, 8256, 96), (513, 1056, 9248), (1024, 256, 4096), (1300, 6528, 608), (2100, 4128, 96)]


@gpu
@pytest.mark.parametrize("kind", ["bf16", "fp16", "fp8"])
@pytest.mark.parametrize("m, n, k", OUT8)
def test_mxfp8_outputs_are_those_of_32_bit_sums(m, n, k, kind):
    import flashinfer_amd as fi

    gen = torch.Generator(device="cuda").manual_seed(m + n + k)
    a, a_scale, a64, at = exact_tokens(m, k, kind, gen)
    b, b_scale, w64 = exact_weights(2 * n, k, at, gen, positive=True)
    g, u = a64 @ w64[:n].T, a64 @ w64[n:].T
    # where exp(-g) vanishes beside 1 in 32 bits, silu(g) is g
    assert g.min() > 40 and max(g.max(), u.abs().max()) < 2 ** 22
    want_q, want_s = to8_bits((g * u).float())
    q, s = fi.gemm_mxfp4_nt_gated(a, b, b_scale, a_scale, out_dtype=FP8)
    assert torch.equal(s, want_s), f"{(s != want_s).sum()} scales of {s.numel()}"
    assert torch.equal(q.view(torch.uint8), want_q)


@gpu
@pytest.mark.parametrize("kind", ["bf16", "fp16"])
@pytest.mark.parametrize("m, n, k", [(1, 70, 6176), (16, 33, 4096), (20, 2001, 1056), (64, 5003, 416),
                                     (70, 6100, 1056), (100, 4256, 1056), (130, 301, 544),
                                     (513, 608, 9248), (1300, 13002, 608)])
def test_16_bit_products_are_those_of_32_bit_sums(m, n, k, kind):
    import flashinfer_amd as fi

    gen = torch.Generator(device="cuda").manual_seed(m + n + k)
    a, _, a64, at = exact_tokens(m, k, kind, gen)
    b, b_scale, w64 = exact_weights(n, k, at, gen, positive=False)
    want = (a64 @ w64.T).to(a.dtype)
    assert want.isfinite().all()
    assert torch.equal(fi.gemm_mxfp4_nt(a, b, b_scale), want)


@gpu
def test_norm_takes_eps_in_64_bits():
    """0.1 is no float32: rounded to one it is off by 1.5e-8, enough to take a value
    next to the border of two scales over it."""
    import flashinfer_amd as fi

    from test_mx import norm64

    eps = 0.1
    w = (100 * (1 + torch.arange(64, device="cuda") * 2.0 ** -20)).float().repeat_interleave(BLOCK)
    # where 100 c / sqrt(c^2 + eps) is 1.75, and a thousand steps around it
    middle = 1.75 * (eps / (100 ** 2 - 1.75 ** 2)) ** 0.5
    start = torch.tensor(middle, device="cuda").view(torch.int32) - 1600
    c = (start + torch.arange(2048, dtype=torch.int32, device="cuda")).view(torch.float32)
    x = c[:, None].expand(2048, 2048).contiguous()
    _, s = fi.rmsnorm_mxfp8_quant(x, w, eps=eps)

    def scales(e):
        return torch.where(norm64(x, w, e)[:, ::BLOCK] > 1.75, 120, 119).to(torch.uint8)

    want = scales(eps)
    assert not torch.equal(want, scales(torch.tensor(eps).item())), "no value that eps decides"
    assert torch.equal(s, want)


def power64(e):
    """2^e in 64 bits from its bits (torch.ldexp takes a power of 32, and a GPU's is
    not always exact)."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def scale_operands(m, n, k, kind):
    """Tokens and weights of every size: row i of b has the scale byte 254 * i // (n - 1),
    token i is about as large as the inverse of byte 254 * i // (m - 1)."""
    gen = torch.Generator(device="cuda").manual_seed(m + n + k)
    b_byte = torch.arange(n, device="cuda") * 254 // (n - 1)
    code = torch.randint(1, 8, (n, k), device="cuda", generator=gen)
    code[b_byte == 253] = code[b_byte == 253].clamp(max=5)  # 3: 4 * 2^126 is no float32
    code[b_byte == 254] = code[b_byte == 254].clamp(max=3)  # 1.5
    b = (code[:, 0::2] | code[:, 1::2] << 4).to(torch.uint8)
    b_scale = b_byte.to(torch.uint8)[:, None].repeat(1, k // BLOCK)
    v = 1 + torch.randint(0, 2, (m, k), device="cuda", generator=gen).double() / 2
    power = 127 - torch.arange(m, device="cuda") * 254 // (m - 1)
    if kind == "fp16":
        power = power.clamp(-15, 14)
    a64 = v * power64(power)[:, None]
    if kind == "fp8":
        a, a_scale = v.float().to(FP8), (power + 127).to(torch.uint8)[:, None].repeat(1, k // BLOCK)
    else:
        a, a_scale = a64.to(KINDS[kind]), None
        assert torch.equal(a.double(), a64)
    ones = torch.full_like(b_scale, 127)
    return a, a_scale, a64, b, b_scale, from4(b, ones) * power64(b_byte - 127)[:, None]


@gpu
@pytest.mark.parametrize("kind", ["bf16", "fp16", "fp8"])
@pytest.mark.parametrize("m, n, k", [(12, 255, 160), (60, 509, 96), (255, 300, 160), (400, 33000, 160)])
def test_every_scale_byte(m, n, k, kind):
    """Scales from 2^-127 to 2^127 on either side. Values from 1 to 6 leave every sum
    exact, and no two of its products are far apart."""
    import flashinfer_amd as fi

    a, a_scale, a64, b, b_scale, w64 = scale_operands(m, n, k, kind)
    want = (a64 @ w64.T).to(torch.bfloat16)
    out = fi.gemm_mxfp4_nt(a, b, b_scale, a_scale, out_dtype=torch.bfloat16)
    # results below the least normal number apart
    seen = want.abs() >= 2.0 ** -126
    assert seen.float().mean() > 0.4 and torch.equal(out[seen], want[seen])
    assert (out[~seen].abs() <= 2.0 ** -126).all()


@gpu
@pytest.mark.parametrize("kind", ["bf16", "fp16", "fp8"])
@pytest.mark.parametrize("m, n, k", [(12, 256, 160), (60, 512, 96), (255, 320, 160), (400, 16512, 160)])
def test_every_scale_byte_and_mxfp8_outputs(m, n, k, kind):
    import flashinfer_amd as fi

    a, a_scale, a64, b, b_scale, w64 = scale_operands(m, n, k, kind)
    b, b_scale, w64 = torch.cat((b, b)), torch.cat((b_scale, b_scale)), torch.cat((w64, w64))
    g = a64 @ w64[:n].T
    # silu(g) is g in 32 bits from about 20 on
    y = (g * g).float()
    plain = ((g > 20) & y.isfinite()).unflatten(1, (-1, BLOCK)).all(-1)
    assert plain.float().mean() > 0.02
    want_q, want_s = to8_bits(y)
    q, s = fi.gemm_mxfp4_nt_gated(a, b, b_scale, a_scale, out_dtype=FP8)
    assert torch.equal(s[plain], want_s[plain])
    q, want_q = (t.view(torch.uint8).unflatten(1, (-1, BLOCK)) for t in (q, want_q))
    assert torch.equal(q[plain], want_q[plain])


@gpu
@pytest.mark.parametrize("kind", ["bf16", "fp16", "fp8"])
@pytest.mark.parametrize("m", [4, 40, 100, 300])
def test_weights_of_2_to_the_128(m, kind):
    """What 16 bits do not hold is not finite, and nothing beside it is touched;
    MXFP8 tokens take the scale as it is."""
    import flashinfer_amd as fi

    n, k = 64, 64
    b = torch.zeros(n, k // 2, dtype=torch.uint8, device="cuda")
    b_scale = torch.full((n, k // BLOCK), 127, dtype=torch.uint8, device="cuda")
    b[:, 0] = 7
    b[3, 0], b[4, 0], b[5, 0] = 6, 5, 3  # 4, 3 and 1.5
    b_scale[:6, 0] = torch.tensor([252, 253, 254, 253, 253, 254], device="cuda")
    a, a_scale = torch.full((m, k), 2.0 ** -14, device="cuda"), None
    if kind == "fp8":
        a, a_scale = fi.mxfp8_quantize(a)
    else:
        a = a.to(KINDS[kind])
    level = torch.tensor([6, 6, 6, 4, 3, 1.5] + [6] * 58, device="cuda", dtype=torch.float64)
    want = (level * power64(b_scale[:, 0].long() - 127) * 2.0 ** -14).to(torch.bfloat16)
    out = fi.gemm_mxfp4_nt(a, b, b_scale, a_scale, out_dtype=torch.bfloat16)
    past = torch.zeros(n, dtype=torch.bool, device="cuda")
    past[1:4] = kind != "fp8"
    assert torch.equal(out[:, ~past], want[~past].expand(m, -1))
    assert not out[:, past].isfinite().any()


@gpu
def test_norms_of_one_dimension_and_of_more_rows_than_a_launch():
    """A row alone, and 2^21 rows and some, which go in two launches, inside wider
    tensors: input, residual and outputs advance by their own strides."""
    import flashinfer_amd as fi

    k, rows = 64, 2 ** 21 + 5
    w = torch.linspace(0.5, 2, k, device="cuda").bfloat16()
    wide = torch.randn(7, 3 * k, device="cuda").bfloat16().repeat(rows // 7 + 1, 1)[:rows]
    x, r = wide[:, :k], wide[:, k + 8:2 * k + 8]
    few_x, few_r = x[:7].clone(), r[:7].clone()
    beside = wide[:, 2 * k + 8:].clone()
    want_q, want_s = fi.fused_add_rmsnorm_mxfp8_quant(few_x, few_r, w)
    q, s = fi.fused_add_rmsnorm_mxfp8_quant(x, r, w)
    for i in range(7):
        assert bool((q[i::7].view(torch.uint8) == want_q[i].view(torch.uint8)).all())
        assert bool((s[i::7] == want_s[i]).all()) and bool((r[i::7] == few_r[i]).all())
    assert torch.equal(wide[:, 2 * k + 8:], beside)
    for f in (fi.mxfp8_quantize, lambda t: fi.rmsnorm_mxfp8_quant(t, w)):
        (q, s), (want_q, want_s) = f(few_x[2]), f(few_x)
        assert q.shape == (k,) and s.shape == (k // BLOCK,)
        assert torch.equal(q.view(torch.uint8), want_q[2].view(torch.uint8))
        assert torch.equal(s, want_s[2])
