"""Every kernel that an MXFP4 product can get, whole and in parts of K: the sizes
below reach each of them for each type and form, which a test without a GPU holds
against the choice itself."""
import math
import random

import pytest
import torch

from flashinfer_amd._lib import get_ext, has_ext
from test_mx import (FP8, OUT_HALF, act64, activations, from4, gpu, product_off, to8_bits, weights4)
from test_mx_sums import exact_tokens, exact_weights

BF16 = torch.bfloat16
# type of a, of the output, gated
FORMS = {"16 bits": (BF16, BF16, False), "MXFP8": (FP8, BF16, False),
         "gated, 16 bits": (BF16, BF16, True), "gated, 16 bits to MXFP8": (BF16, FP8, True),
         "gated, MXFP8 to 16 bits": (FP8, BF16, True), "gated, MXFP8": (FP8, FP8, True)}
PLAIN = [(1, 33, 32), (34, 33, 32), (65, 37, 2752), (4164, 67, 32), (20, 16905, 32), (34, 17448, 32),
         (67, 16830, 32), (261, 22424, 32), (2093, 33, 7072), (65, 18853, 480), (92, 2066, 7360),
         (4828, 77, 6112), (2889, 74, 11360), (4244, 92, 14240), (5577, 340, 7584), (215, 17423, 13728),
         (66, 16961, 3200), (342, 3170, 13184), (223, 10402, 8960), (1788, 2434, 13248)]
GATED = [(1, 32, 32), (81, 4192, 32), (33, 10400, 32), (65, 8544, 32), (40, 8800, 192), (72, 1440, 8352),
         (65, 12256, 1120), (274, 17760, 288), (163, 1056, 11712), (255, 1056, 14176), (115, 8416, 8672),
         (1925, 544, 9056), (71, 18144, 15200), (890, 2112, 4352), (2164, 1056, 9216), (4145, 96, 96),
         (70, 96, 4128), (70, 96, 96), (260, 320, 6176), (100, 4256, 13056)]


def chosen(form, m, n, k):
    name, parts = get_ext().gemm_mxfp4_plan(*FORMS[form], m, n, k)
    return name, parts > 1


@pytest.mark.skipif(not has_ext(), reason="native extension not built")
@pytest.mark.parametrize("form", FORMS)
def test_the_sizes_reach_every_kernel(form):
    rng = random.Random(0)

    def size(most):
        return round(math.exp(rng.uniform(0, math.log(most))))

    reached = {chosen(form, size(8192), 32 * size(1024), 32 * size(512)) for _ in range(40000)}
    assert len(reached) > 10
    missing = reached - {chosen(form, *s) for s in (GATED if FORMS[form][2] else PLAIN)}
    assert not missing, f"no size for {sorted(missing)}"


@gpu
@pytest.mark.parametrize("kind", ["bf16", "fp16", "fp8"])
@pytest.mark.parametrize("m, n, k", PLAIN)
def test_plain(m, n, k, kind):
    import flashinfer_amd as fi

    gen = torch.Generator(device="cuda").manual_seed(m + n + k)
    if kind == "fp8":
        a, a_scale, a64 = activations(m, k, kind, gen)
        b, b_scale = weights4(n, k, gen)
        w64 = from4(b, b_scale)
        want, off = a64 @ w64.T, product_off(a64, w64, kind)
        for dtype in (torch.bfloat16, torch.float16):
            out = fi.gemm_mxfp4_nt(a, b, b_scale, a_scale, out_dtype=dtype)
            # fp16 has a least step of 2^-24
            bound = off + OUT_HALF[dtype] * (want.abs() + off) + 2.0 ** -25
            assert ((out.double() - want).abs() <= bound).all()
    else:
        a, a_scale, a64, at = exact_tokens(m, k, kind, gen)
        b, b_scale, w64 = exact_weights(n, k, at, gen, positive=False)
        want = a64 @ w64.T
        for dtype in (torch.bfloat16, torch.float16):
            assert torch.equal(fi.gemm_mxfp4_nt(a, b, b_scale, out_dtype=dtype), want.to(dtype))


@gpu
@pytest.mark.parametrize("kind", ["bf16", "fp16", "fp8"])
@pytest.mark.parametrize("m, n, k", GATED)
def test_gated(m, n, k, kind):
    import flashinfer_amd as fi

    gen = torch.Generator(device="cuda").manual_seed(m + n + k)
    a, a_scale, a64, at = exact_tokens(m, k, kind, gen)
    b, b_scale, w64 = exact_weights(2 * n, k, at, gen, positive=True)
    # silu(g) is g in 32 bits where exp(-g) vanishes beside 1
    g, u = a64 @ w64[:n].T, a64 @ w64[n:].T
    assert g.min() > 20 and max(g.max(), u.abs().max()) < 2 ** 22
    y = (g * u).float()
    want_q, want_s = to8_bits(y)
    q, s = fi.gemm_mxfp4_nt_gated(a, b, b_scale, a_scale, out_dtype=FP8)
    assert torch.equal(s, want_s) and torch.equal(q.view(torch.uint8), want_q)
    if kind != "fp8":
        assert torch.equal(fi.gemm_mxfp4_nt_gated(a, b, b_scale, out_dtype=BF16), y.to(BF16))
        return
    a, a_scale, a64 = activations(m, k, kind, gen)
    b, b_scale = weights4(2 * n, k, gen)
    w64 = from4(b, b_scale)
    g, u = a64 @ w64[:n].T, a64 @ w64[n:].T
    og, ou = product_off(a64, w64[:n], kind), product_off(a64, w64[n:], kind)
    want = act64(g, "silu") * u
    og = 1.13 * og + 8 * 2.0 ** -24 * g.abs()
    off = og * (u.abs() + ou) + act64(g, "silu").abs() * ou
    out = fi.gemm_mxfp4_nt_gated(a, b, b_scale, a_scale, out_dtype=BF16)
    assert ((out.double() - want).abs() <= off + 2.0 ** -8 * (want.abs() + off)).all()


@gpu
@pytest.mark.parametrize("kind", ["bf16", "fp16", "fp8"])
@pytest.mark.parametrize("m", [70, 97])
def test_rows_too_far_apart_for_32_bits(m, kind):
    """Rows 16 MB apart go 16 tokens at a time through the kernel for few tokens,
    with their own scales, outputs and output scales; so do outputs far apart."""
    import flashinfer_amd as fi

    gen = torch.Generator(device="cuda").manual_seed(m)
    n, k = 96, 288
    a, a_scale, a64, at = exact_tokens(m, k, kind, gen)
    b, b_scale, w64 = exact_weights(2 * n, k, at, gen, positive=True)
    far = torch.empty(m, (1 << 24) // a.element_size() + 16, dtype=a.dtype, device="cuda")[:, :k]
    far.copy_(a)
    if kind == "fp8":
        # scales of its own for every row, within what 32 bits add up exactly
        a_scale += (torch.arange(m, device="cuda") % 5).to(torch.uint8)[:, None]
        a64 = a64 * 2.0 ** (torch.arange(m, device="cuda") % 5)[:, None]
    g, u = a64 @ w64[:n].T, a64 @ w64[n:].T
    want_q, want_s = to8_bits((g * u).float())
    assert len({tuple(r) for r in want_s.tolist()}) > 1
    q, s = fi.gemm_mxfp4_nt_gated(far, b, b_scale, a_scale, out_dtype=FP8)
    assert torch.equal(s, want_s) and torch.equal(q.view(torch.uint8), want_q)
    box = torch.empty(m, n + 40, dtype=torch.uint8, device="cuda").view(FP8)[:, :n]
    q, s = fi.gemm_mxfp4_nt_gated(far, b, b_scale, a_scale, out=box)
    assert torch.equal(s, want_s) and torch.equal(q.view(torch.uint8), want_q)
    out = fi.gemm_mxfp4_nt(far, b, b_scale, a_scale, out_dtype=BF16)
    if kind == "fp8":
        want, off = a64 @ w64.T, product_off(a64, w64, kind)
        assert ((out.double() - want).abs() <= off + 2.0 ** -8 * (want.abs() + off)).all()
    else:
        assert torch.equal(out, (a64 @ w64.T).to(BF16))


@gpu
@pytest.mark.parametrize("kind", ["bf16", "fp16", "fp8"])
@pytest.mark.parametrize("m, n, k", [(1, 64, 32), (7, 7008, 160), (12, 96, 6176), (30, 64, 288)] + GATED[1:])
def test_special_values_and_mxfp8_outputs(m, n, k, kind):
    """A NaN or an infinity makes the blocks NaN that it reaches and leaves the others
    as they were, bit by bit."""
    import flashinfer_amd as fi

    gen = torch.Generator(device="cuda").manual_seed(m + n + k)
    a, a_scale, _, at = exact_tokens(m, k, kind, gen)
    b, b_scale, _ = exact_weights(2 * n, k, at, gen, positive=True)

    def run():
        q, s = fi.gemm_mxfp4_nt_gated(a, b, b_scale, a_scale, out_dtype=FP8)
        return q.view(torch.uint8).unflatten(1, (-1, 32)), s

    q0, s0 = run()
    assert (s0 < 255).all()
    bad = torch.zeros(m, n // 32, dtype=torch.bool, device="cuda")
    gate, up, last = n // 2, n + n - 1, k // 32 - 1
    b_scale[gate, last] = 255
    b[up, :16] = 0  # NaN times zero
    b_scale[up, 0] = 255
    bad[:, gate // 32] = bad[:, -1] = True
    if m > 2:
        if kind == "fp8":
            a_scale[m // 2, last] = 255
            a_scale[m - 1, 0] = 255
            a.view(torch.uint8)[m - 1, :32] = 0
        else:
            a[m // 2, k - 1] = math.nan
            a[m - 1, 3] = math.inf
        bad[m // 2] = bad[m - 1] = True
    q, s = run()
    assert torch.equal(s == 255, bad)
    assert (q[bad] & 0x7F == 0x7F).all()
    assert torch.equal(s[~bad], s0[~bad]) and torch.equal(q[~bad], q0[~bad])


@gpu
def test_more_tiles_than_one_launch():
    """Tiles of more than 2^32 threads: 547 x 32768 of 128 x 128 with 256 lanes each."""
    import flashinfer_amd as fi

    torch.cuda.empty_cache()
    m, n, k = 70000, 2 ** 21, 32
    assert chosen("gated, MXFP8", m, n, k) == ("128x128", False)
    gen = torch.Generator(device="cuda").manual_seed(0)
    a, a_scale, _, at = exact_tokens(m, k, "fp8", gen)
    few, few_scale, _ = exact_weights(64, k, at, gen, positive=True)
    b = torch.zeros(2 * n, k // 2, dtype=torch.uint8, device="cuda")
    b_scale = torch.full((2 * n, k // 32), 127, dtype=torch.uint8, device="cuda")
    b[n - 32:n], b[-32:] = few[:32], few[32:]
    want_q, want_s = fi.gemm_mxfp4_nt_gated(a, few, few_scale, a_scale, out_dtype=FP8)
    q, s = fi.gemm_mxfp4_nt_gated(a, b, b_scale, a_scale, out_dtype=FP8)
    assert torch.equal(s[:, -1:], want_s) and not s[:, :-1].any()
    assert torch.equal(q[:, -32:].view(torch.uint8), want_q.view(torch.uint8))
    for at in range(0, m, 10000):
        assert not q[at:at + 10000, :-32].view(torch.uint8).any()
    del q, s
    torch.cuda.empty_cache()


@gpu
@pytest.mark.parametrize("m", [3, 40, 300])
def test_scales_as_float8_e8m0fnu(m):
    import flashinfer_amd as fi

    a, a_scale, _ = activations(m, 160, "fp8")
    b, b_scale = weights4(192, 160)
    e8m0 = torch.float8_e8m0fnu
    want = fi.gemm_mxfp4_nt(a, b, b_scale, a_scale)
    assert torch.equal(fi.gemm_mxfp4_nt(a, b, b_scale.view(e8m0), a_scale.view(e8m0)), want)
    want_q, want_s = fi.gemm_mxfp4_nt_gated(a, b, b_scale, a_scale, out_dtype=FP8)
    q, s = fi.gemm_mxfp4_nt_gated(a, b, b_scale.view(e8m0), a_scale.view(e8m0), out_dtype=FP8)
    assert torch.equal(s, want_s) and torch.equal(q.view(torch.uint8), want_q.view(torch.uint8))
