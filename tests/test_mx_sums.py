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
