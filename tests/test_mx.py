"""MX formats: RMSNorm and activations written as MXFP8, products with MXFP4
weights (plain and gated). Every result is held to the definition in 64 bits.

Tolerances, from the arithmetic:
  * an output in type t rounds by at most half a step, ``eps(t) / 2`` of its
    value; e4m3 also by half of its smallest step, 2^-10 of its scale;
  * a sum of n products held in 32 bits is off by at most n * 2^-24 of the sum
    of their magnitudes;
  * an instruction on 8-bit operands aligns its 128 products to the largest of
    them and keeps 18 bits below it, so its sum is off by at most 128 * 2^-18 =
    2^-11 of the sum of the magnitudes.
"""
import math

import pytest
import torch

from flashinfer_amd._lib import has_ext

gpu = pytest.mark.gpu
FP8 = torch.float8_e4m3fn
BLOCK = 32
E4M3_HALF = 2.0 ** -4
OUT_HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
LEVELS = [0, 0.5, 1, 1.5, 2, 3, 4, 6, -0.0, -0.5, -1, -1.5, -2, -3, -4, -6]


def scale64(byte):
    s = torch.ldexp(torch.ones(byte.shape, dtype=torch.float64, device=byte.device),
                    byte.to(torch.int64) - 127)
    return torch.where(byte == 255, torch.full_like(s, math.nan), s)


def from8(q, scale):
    s = scale64(scale.view(torch.uint8)).repeat_interleave(BLOCK, -1)
    return q.view(FP8).to(torch.float64) * s


def from4(packed, scale):
    levels = torch.tensor(LEVELS, dtype=torch.float64, device=packed.device)
    code = torch.stack((packed & 15, packed >> 4), -1).flatten(-2).long()
    return levels[code] * scale64(scale.view(torch.uint8)).repeat_interleave(BLOCK, -1)


def act64(g, name):
    if name == "silu":
        return g * torch.sigmoid(g)
    if name == "gelu":
        return g * torch.special.ndtr(g)
    return g * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (g + 0.044715 * g ** 3))


def check8(q, scale, y, off):
    """q, scale against the 64-bit y, which the kernel may miss by ``off``
    before it rounds."""
    blocks = y.unflatten(-1, (-1, BLOCK))
    most, slack = blocks.abs().amax(-1), off.unflatten(-1, (-1, BLOCK)).amax(-1)
    s = scale64(scale)
    # the least power of two with which nothing saturates, but for a maximum
    # so near to a border that ``off`` decides
    assert (448 * s >= most - slack).all(), "a block saturates"
    low = scale > 0
    assert (224 * s < most + slack)[low].all(), "a scale is larger than it has to be"
    wide = s.repeat_interleave(BLOCK, -1)
    err = (from8(q, scale) - y).abs()
    bound = off * (1 + E4M3_HALF) + E4M3_HALF * y.abs() + 2.0 ** -10 * wide
    assert (err <= bound).all(), f"off by {(err / bound).max()} of the bound"


def weights4(n, k, gen=None, spread=3):
    dev = "cuda"
    w = torch.randint(0, 256, (n, k // 2), dtype=torch.uint8, device=dev, generator=gen)
    # exponents around that of 1 / sqrt(k)
    mid = 127 - 2 - int(math.log2(k) / 2)
    s = torch.randint(mid - spread, mid + spread + 1, (n, k // BLOCK), device=dev,
                      generator=gen).to(torch.uint8)
    return w, s


def activations(m, k, kind, gen=None):
    """(what the call takes, its scale or None, its values in 64 bits)"""
    import flashinfer_amd as fi

    x = torch.randn(m, k, device="cuda", generator=gen)
    x[:, ::17] *= 8
    if kind == "fp8":
        q, s = fi.mxfp8_quantize(x)
        return q, s, from8(q, s)
    x = x.to({"bf16": torch.bfloat16, "fp16": torch.float16}[kind])
    return x, None, x.double()


def product_off(a64, w64, kind):
    """How far a product may be off before it is rounded to the output's type."""
    rel = 2.0 ** -11 if kind == "fp8" else a64.shape[1] * 2.0 ** -24
    if kind == "fp16":
        rel = 2 * rel  # two products where a is split
    return rel * (a64.abs() @ w64.abs().T)


# ------------------------------------------------------------ weights, on the CPU

def test_mxfp4_quantize_is_nearest():
    from flashinfer_amd import mxfp4_quantize

    gen = torch.Generator().manual_seed(0)
    w = torch.randn(7, 96, generator=gen) * torch.exp2(torch.randint(-9, 9, (7, 1), generator=gen))
    b, s = mxfp4_quantize(w)
    assert b.shape == (7, 48) and s.shape == (7, 3)
    got = from4(b, s)
    sc = scale64(s).repeat_interleave(BLOCK, -1)
    levels = torch.tensor(LEVELS, dtype=torch.float64)
    best = (w.double().unsqueeze(-1) - levels * sc.unsqueeze(-1)).abs().amin(-1)
    torch.testing.assert_close((got - w.double()).abs(), best, rtol=0, atol=0)
    most = w.double().abs().unflatten(-1, (-1, BLOCK)).amax(-1)
    assert (6 * scale64(s) >= most).all() and (3 * scale64(s) < most).all()


def test_mxfp4_quantize_ties_go_to_the_even_code():
    from flashinfer_amd import mxfp4_quantize

    w = torch.zeros(2, 32)
    w[0, :8] = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0])
    w[1] = -w[0]
    b, s = mxfp4_quantize(w)
    assert (s == 127).all()
    want = torch.tensor([0, 1, 1, 2, 2, 4, 4, 6], dtype=torch.float64)
    assert torch.equal(from4(b, s)[0, :8], want)
    assert torch.equal(from4(b, s)[1, :8], -want)


def test_mxfp4_quantize_special_blocks():
    from flashinfer_amd import mxfp4_quantize

    w = torch.ones(4, 64)
    w[0, 3], w[1, 40], w[2, :32] = math.nan, math.inf, 0
    w[3, :32] = 6e-39  # below the least normal number: 2^-127 is 5.9e-39
    b, s = mxfp4_quantize(w)
    d = from4(b, s)
    assert d[0, :32].isnan().all() and (d[0, 32:] == 1).all()
    assert d[1, 32:].isnan().all() and (d[1, :32] == 1).all()
    assert (d[2, :32] == 0).all() and s[3, 0] == 0 and (d[3, :32] > 0).all()


@pytest.mark.parametrize("shape", [(32,), (4, 0), (4, 48)])
def test_mxfp4_quantize_refuses(shape):
    from flashinfer_amd import mxfp4_quantize

    with pytest.raises(ValueError):
        mxfp4_quantize(torch.zeros(shape))


# ------------------------------------------------------------ refusals, on the CPU

def _operands(m=4, n=64, k=64, dtype=torch.bfloat16):
    return [torch.zeros(m, k, dtype=dtype), torch.zeros(n, k // 2, dtype=torch.uint8),
            torch.zeros(n, k // 32, dtype=torch.uint8)]


needs_ext = pytest.mark.skipif(not has_ext(), reason="native extension not built")


@needs_ext
@pytest.mark.parametrize("what, change", [
    ("two-dimensional", lambda o: o.__setitem__(0, o[0][0])),
    ("a is bfloat16", lambda o: o.__setitem__(0, o[0].float())),
    ("multiple of 32", lambda o: o.__setitem__(0, o[0][:, :48])),
    ("multiple of 32", lambda o: o.__setitem__(0, o[0][:, :0])),
    ("b must be contiguous", lambda o: o.__setitem__(1, o[1][:, :16])),
    ("b must be contiguous", lambda o: o.__setitem__(1, o[1].to(torch.int8))),
    ("b must be contiguous", lambda o: o.__setitem__(1, torch.zeros(64, 64, dtype=torch.uint8)[:, :32])),
    ("b_scale must be", lambda o: o.__setitem__(2, o[2][:1])),
    ("b_scale must be", lambda o: o.__setitem__(2, o[2].float())),
    ("a_scale belongs", lambda o: o.append(torch.zeros(4, 2, dtype=torch.uint8))),
    ("a_scale belongs", lambda o: o.__setitem__(0, torch.zeros(4, 64).to(FP8))),
    ("a_scale must be", lambda o: (o.__setitem__(0, torch.zeros(4, 64).to(FP8)),
                                   o.append(torch.zeros(3, 2, dtype=torch.uint8)))),
    ("rows of a", lambda o: o.__setitem__(0, torch.zeros(64, 4, dtype=torch.bfloat16).t())),
    ("rows of a", lambda o: o.__setitem__(0, torch.zeros(4, 68, dtype=torch.bfloat16)[:, :64])),
    ("rows of a", lambda o: o.__setitem__(0, torch.zeros(264, dtype=torch.bfloat16)[1:257].view(4, 64))),
    ("rows of a", lambda o: o.__setitem__(0, torch.zeros(1, 64, dtype=torch.bfloat16).expand(4, 64))),
    ("must be on a GPU", lambda o: None),
])
@pytest.mark.parametrize("gated", [False, True])
def test_product_refusals(what, change, gated):
    import flashinfer_amd as fi

    o = _operands()
    change(o)
    with pytest.raises(ValueError, match=what):
        (fi.gemm_mxfp4_nt_gated if gated else fi.gemm_mxfp4_nt)(*o)


@needs_ext
@pytest.mark.parametrize("m, n, k", [(1, 2 ** 26 + 2, 32), (1, 2, 2 ** 29 + 32)])
def test_sizes_past_a_launch_are_refused(m, n, k):
    import flashinfer_amd as fi

    o = [torch.empty(m, k, dtype=torch.bfloat16), torch.empty(n, k // 2, dtype=torch.uint8),
         torch.empty(n, k // 32, dtype=torch.uint8)]
    for f in (fi.gemm_mxfp4_nt, fi.gemm_mxfp4_nt_gated):
        with pytest.raises(ValueError, match="the rows of b to"):
            f(*o)


@needs_ext
@pytest.mark.parametrize("what, kw", [
    ("out is bfloat16", dict(out_dtype=torch.float32)),
    ("out is bfloat16", dict(out_dtype=FP8)),
    ("out must be", dict(out=torch.zeros(4, 63, dtype=torch.bfloat16))),
    ("out must be", dict(out=torch.zeros(4, 64, dtype=torch.float16), out_dtype=torch.bfloat16)),
    ("rows of out", dict(out=torch.zeros(64, 4, dtype=torch.bfloat16).t())),
    ("rows of out", dict(out=torch.zeros(1, 64, dtype=torch.bfloat16).expand(4, 64))),
])
def test_gemm_output_refusals(what, kw):
    import flashinfer_amd as fi

    with pytest.raises(ValueError, match=what):
        fi.gemm_mxfp4_nt(*_operands(), **kw)


@needs_ext
@pytest.mark.parametrize("what, n, kw", [
    ("activation is one of", 64, dict(activation="relu")),
    ("as many up rows", 63, {}),
    ("multiple of 32", 96, dict(out_dtype=FP8)),
    ("out_scale belongs", 64, dict(out_scale=torch.zeros(4, 1, dtype=torch.uint8))),
    ("out_scale must be", 64, dict(out_dtype=FP8, out_scale=torch.zeros(4, 2, dtype=torch.uint8))),
    ("multiples of 8 bytes", 64, dict(out=torch.zeros(4, 36).to(FP8)[:, :32])),
])
def test_gated_refusals(what, n, kw):
    import flashinfer_amd as fi

    with pytest.raises(ValueError, match=what):
        fi.gemm_mxfp4_nt_gated(*_operands(n=n), **kw)


@needs_ext
@pytest.mark.parametrize("what, args, kw", [
    ("multiple of 32", (torch.zeros(2, 48), torch.zeros(48)), {}),
    ("multiple of 32", (torch.zeros(2, 65568), torch.zeros(65568)), {}),
    ("last dimension", (torch.zeros(()), torch.zeros(1)), {}),
    ("the input is", (torch.zeros(2, 64).double(), torch.zeros(64).double()), {}),
    ("weight must be", (torch.zeros(2, 64), torch.zeros(32)), {}),
    ("weight must be", (torch.zeros(2, 64), torch.zeros(64).half()), {}),
    ("the input must be contiguous", (torch.zeros(64, 2).t(), torch.zeros(64)), {}),
    ("the input must be contiguous", (torch.zeros(2, 2, 128)[:, :, :64], torch.zeros(64)), {}),
    ("out must be", (torch.zeros(2, 64), torch.zeros(64)), dict(out=torch.zeros(2, 64))),
    ("out_scale must be", (torch.zeros(2, 64), torch.zeros(64)),
     dict(out_scale=torch.zeros(2, 64, dtype=torch.uint8))),
    ("must be on a GPU", (torch.zeros(2, 64), torch.zeros(64)), {}),
])
def test_norm_refusals(what, args, kw):
    import flashinfer_amd as fi

    with pytest.raises(ValueError, match=what):
        fi.rmsnorm_mxfp8_quant(*args, **kw)
    x, w = args
    with pytest.raises(ValueError, match=what):
        fi.fused_add_rmsnorm_mxfp8_quant(x, x.clone(), w, **kw)


@needs_ext
def test_residual_refusals():
    import flashinfer_amd as fi

    x, w = torch.zeros(2, 64), torch.zeros(64)
    for r in (torch.zeros(1, 64), torch.zeros(2, 64).half()):
        with pytest.raises(ValueError, match="the residual must have"):
            fi.fused_add_rmsnorm_mxfp8_quant(x, r, w)
    with pytest.raises(ValueError, match="the residual must be contiguous"):
        fi.fused_add_rmsnorm_mxfp8_quant(x, torch.zeros(64, 2).t(), w)


@gpu
def test_overlapping_operands_are_refused():
    import flashinfer_amd as fi

    x = torch.zeros(4, 64, dtype=torch.bfloat16, device="cuda")
    w = torch.zeros(64, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(ValueError, match="share memory"):
        fi.fused_add_rmsnorm_mxfp8_quant(x, x, w)
    with pytest.raises(ValueError, match="share memory"):
        fi.rmsnorm_mxfp8_quant(x, w, out=x.view(torch.uint8).view(-1)[:256].view(4, 64).view(FP8))
    b = torch.zeros(64, 32, dtype=torch.uint8, device="cuda")
    s = torch.zeros(64, 2, dtype=torch.uint8, device="cuda")
    with pytest.raises(ValueError, match="share memory"):
        fi.gemm_mxfp4_nt(x, b, s, out=x)
    with pytest.raises(ValueError, match="operands are on"):
        fi.gemm_mxfp4_nt(x, b.cpu(), s)


# ------------------------------------------------------------ MXFP8 output

def to8_bits(x):
    """x (32-bit) as MXFP8 by whole-number work on its bits."""
    bits = (x.view(torch.int32) & 0x7FFFFFFF).unflatten(-1, (-1, BLOCK)).amax(-1)
    byte = ((bits >> 23) - 8 + ((bits & 0x7FFFFF) > 0x600000).int()).clamp(min=0)
    bad = bits >= 0x7F800000
    byte = torch.where(bad, torch.full_like(byte, 255), byte)
    wide = torch.where(bad, torch.full_like(byte, 127), byte).repeat_interleave(BLOCK, -1)
    q = torch.ldexp(x.double(), 127 - wide).float().to(FP8).view(torch.uint8)
    q = torch.where(bad.repeat_interleave(BLOCK, -1), torch.full_like(q, 0x7F), q)
    return q, byte.to(torch.uint8)


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("rows, k", [(1, 32), (65, 32), (33, 64), (3, 96), (19, 128), (17, 160),
                                     (9, 256), (5, 288), (5, 4096), (2, 8224), (2, 16416), (3, 65536)])
def test_quantize_is_exact(rows, k, dtype):
    import flashinfer_amd as fi

    torch.manual_seed(rows + k)
    x = torch.randn(rows, k, device="cuda")
    x *= torch.exp2(torch.randint(-10, 5, (rows, k // BLOCK), device="cuda")).repeat_interleave(BLOCK, 1)
    x = x.to(dtype)
    q, s = fi.mxfp8_quantize(x)
    assert q.dtype == FP8 and q.shape == (rows, k)
    assert s.dtype == torch.uint8 and s.shape == (rows, k // BLOCK)
    want_q, want_s = to8_bits(x.float())
    assert torch.equal(s, want_s) and torch.equal(q.view(torch.uint8), want_q)


@gpu
def test_quantize_borders_and_special_values():
    import flashinfer_amd as fi

    x = torch.zeros(12, 64, device="cuda")
    x[0, 5] = 448.0                      # the largest value itself
    x[1, 5] = 448.0 * (1 + 2.0 ** -23)   # one step above it
    x[2, 5] = -448.0 * 2.0 ** 100
    x[3, 5] = 3e38
    x[4, 5] = 1e-38
    x[5, 5] = 1e-45                      # the least subnormal
    x[6, 5] = math.inf
    x[7, 5] = math.nan
    x[8, 5], x[8, 6] = -math.inf, 1.0
    x[9, :] = torch.linspace(-17, 31, 64, device="cuda")
    x[10, 5], x[10, 6] = 448.0, 2.0 ** -10  # a tie below the least subnormal e4m3
    x[11, 5], x[11, 6] = 448.0, 1.0625     # a tie between 1 and 1.125
    q, s = fi.mxfp8_quantize(x)
    want_q, want_s = to8_bits(x)
    assert torch.equal(s, want_s) and torch.equal(q.view(torch.uint8), want_q)
    assert s[0, 0] == 127 and s[1, 0] == 128 and s[5, 0] == 0 and s[0, 1] == 0
    for row in (6, 7, 8):
        assert s[row, 0] == 255 and q[row, :32].float().isnan().all()
        assert (q[row, 32:].float() == 0).all()


def norm64(r, w, eps):
    r = r.double()
    return r / torch.sqrt(r.square().mean(-1, keepdim=True) + eps) * w.double()


def norm_off(y, k):
    # the sum of k squares, the root, and three roundings of the products
    return y.abs() * ((k / 2 + 4) * 2.0 ** -24)


@gpu
@pytest.mark.parametrize("add", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("rows, k", [(1, 32), (65, 32), (33, 64), (1, 4096), (7, 96), (19, 128),
                                     (17, 160), (9, 256), (5, 288), (33, 7168), (3, 8224), (2, 65536)])
def test_norm(rows, k, dtype, add):
    import flashinfer_amd as fi

    torch.manual_seed(rows * k)
    x = (torch.randn(rows, k, device="cuda") * 3).to(dtype)
    w = (torch.randn(k, device="cuda") + 1).to(dtype)
    r = torch.randn(rows, k, device="cuda").to(dtype)
    if add:
        want = (x.float() + r.float()).to(dtype)
        q, s = fi.fused_add_rmsnorm_mxfp8_quant(x, r, w, eps=1e-5)
        assert torch.equal(r, want)
    else:
        want = x
        q, s = fi.rmsnorm_mxfp8_quant(x, w, eps=1e-5)
    y = norm64(want, w, 1e-5)
    check8(q, s, y, norm_off(y, k))


@gpu
@pytest.mark.parametrize("k", [128, 4096])
def test_norm_next_to_the_border_of_two_scales(k):
    """Values within 3 steps of 1.75, where the scale changes: roundings of 32 bits
    on the way reach as far, and the scale is that of 64 bits all the same."""
    import flashinfer_amd as fi

    torch.manual_seed(k)
    x = (torch.rand(512, 1, device="cuda") * 1000 + 1000).expand(512, k).contiguous()
    step = torch.arange(k // BLOCK, device="cuda") % 7 - 3
    w = (1.75 + step * 2.0 ** -23).float().repeat_interleave(BLOCK)
    q, s = fi.rmsnorm_mxfp8_quant(x, w)
    # eps takes 1e-13 to 5e-13 away, far more than 64 bits round
    y = norm64(x, w, 1e-6)[:, ::BLOCK]
    assert torch.equal(s, torch.where(y > 1.75, 120, 119).to(torch.uint8))
    # four blocks hold the steps -3 to 0 alone
    assert bool((y < 1.75).any()) and bool((y > 1.75).any()) == (k > 128)


@gpu
def test_norm_of_zero_and_unlike_rows():
    import flashinfer_amd as fi

    x = torch.randn(6, 4096, device="cuda", dtype=torch.bfloat16)
    x[0] = 0
    x[1, 7] = math.nan
    x[2, 7] = math.inf
    x[3] *= 1e-20
    x[4] *= 1e15
    w = torch.ones(4096, device="cuda", dtype=torch.bfloat16)
    w[64:96] = 0
    q, s = fi.rmsnorm_mxfp8_quant(x, w)
    assert (q[0].float() == 0).all() and (s[0] == 0).all()
    assert (s[1] == 255).all() and q[1].float().isnan().all()
    # 1 / inf is 0: the infinity's own block is NaN, the others are 0
    assert s[2, 0] == 255 and (q[2, 32:].float() == 0).all()
    y = norm64(x, w, 1e-6)[3:]
    check8(q[3:], s[3:], y, norm_off(y, 4096))
    assert (from8(q, s)[3:, 64:96] == 0).all()


@gpu
@pytest.mark.parametrize("k", [32, 64, 128, 256])
def test_short_rows_do_not_meet(k):
    import flashinfer_amd as fi

    x = torch.randn(21, k, device="cuda", dtype=torch.bfloat16)
    x[3, 1], x[7, k - 1] = math.nan, 1e30
    w = torch.ones(k, device="cuda", dtype=torch.bfloat16)
    q, s = fi.rmsnorm_mxfp8_quant(x, w)
    assert (s[3] == 255).all()
    rest = [i for i in range(21) if i not in (3, 7)]
    y = norm64(x[rest], w, 1e-6)
    check8(q[rest], s[rest], y, norm_off(y, k))


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_norm_strides_shapes_and_outputs(dtype):
    import flashinfer_amd as fi

    torch.manual_seed(2)
    k = 160
    w = torch.randn(k, device="cuda", dtype=dtype)
    # rows of a wider tensor, at a distance that is no multiple of 16 bytes
    wide = torch.randn(9, 3 * k + 1, device="cuda", dtype=dtype)
    x, r = wide[:, :k], wide[:, k + 1:2 * k + 1]
    kept, want = wide.clone(), (x.float() + r.float()).to(dtype)
    q, s = fi.fused_add_rmsnorm_mxfp8_quant(x, r, w)
    y = norm64(want, w, 1e-6)
    check8(q, s, y, norm_off(y, k))
    kept[:, k + 1:2 * k + 1] = want
    assert torch.equal(wide, kept), "something beside the residual was written"
    # misaligned weight and output
    w1 = torch.cat((w[:1], w))[1:]
    o = torch.zeros(9 * k + 2, dtype=torch.uint8, device="cuda")
    os = torch.zeros(9, k // BLOCK, dtype=torch.uint8, device="cuda")
    got, gs = fi.rmsnorm_mxfp8_quant(want, w1, out=o[1:-1].view(9, k).view(FP8), out_scale=os)
    assert got.data_ptr() == o.data_ptr() + 1 and gs.data_ptr() == os.data_ptr()
    assert torch.equal(got.view(torch.uint8), q.view(torch.uint8)) and torch.equal(os, s)
    assert o[0] == 0 and o[-1] == 0
    # leading dimensions, no rows at all
    q3, s3 = fi.rmsnorm_mxfp8_quant(want.view(3, 3, k), w)
    assert q3.shape == (3, 3, k) and s3.shape == (3, 3, k // BLOCK)
    assert torch.equal(q3.view(torch.uint8).view(9, k), q.view(torch.uint8))
    q0, s0 = fi.rmsnorm_mxfp8_quant(want[:0], w)
    assert q0.shape == (0, k) and s0.shape == (0, k // BLOCK)


# ------------------------------------------------------------ products

SHAPES = [(1, 1, 32), (1, 64, 4096), (3, 17, 160), (16, 100, 512), (17, 33, 1056), (33, 257, 96),
          (64, 48, 2080), (65, 130, 4096), (130, 301, 544), (257, 513, 1024), (1024, 260, 288)]


# tiles with edges on every side, whole and in parts of K
TILES = [(24, 25000, 64), (20, 100, 9248), (40, 300, 8480), (200, 3100, 288), (33, 20500, 160),
         (100, 21000, 96), (520, 8450, 96), (1300, 13002, 608), (100, 8200, 96), (70, 8200, 96),
         (70, 6100, 1056)]
# and every tile again, whole and in parts of K, with 70 tokens or more
EVERY = [(70, 96, 96), (70, 96, 4128), (100, 4256, 96), (100, 8480, 96), (70, 16512, 96),
         (390, 16512, 96), (100, 1056, 6176), (70, 2080, 9248), (70, 8480, 96), (513, 608, 9248),
         (100, 4256, 1056), (70, 16512, 544), (100, 8480, 9248)]
EVERY_GATED = [(70, 96, 96), (100, 2080, 96), (70, 96, 4128), (100, 4256, 96), (200, 4256, 96),
               (130, 16512, 96), (260, 320, 6176), (70, 1056, 9248), (100, 8480, 1056),
               (100, 2080, 9248), (70, 4256, 96), (100, 2080, 14336), (513, 1056, 9248),
               (513, 1056, 14336), (70, 8480, 14336)]


# the kernel for few tokens: K in one, two and three slabs of scales, and the
# three ways to share it
FEW = [(1, 70, 12320), (5, 40, 6176), (16, 33, 14336), (3, 16500, 6240), (2, 7001, 96), (9, 7000, 6144),
       (8, 33, 14336), (6, 7001, 96), (7, 16500, 160)]
# the same with 17 to 32 tokens and 33 to 64
MORE = [(20, 2001, 6240), (32, 5000, 6176), (17, 16600, 160), (32, 4100, 96), (40, 4090, 6176),
        (64, 5003, 416), (33, 17000, 96), (64, 4113, 6176)]


@gpu
@pytest.mark.parametrize("kind", ["bf16", "fp16", "fp8"])
@pytest.mark.parametrize("m, n, k", SHAPES + TILES + EVERY + FEW + MORE)
def test_gemm(m, n, k, kind):
    import flashinfer_amd as fi

    torch.manual_seed(m * n + k)
    a, a_scale, a64 = activations(m, k, kind)
    b, b_scale = weights4(n, k)
    w64 = from4(b, b_scale)
    want, off = a64 @ w64.T, product_off(a64, w64, kind)
    out = fi.gemm_mxfp4_nt(a, b, b_scale, a_scale)
    assert out.shape == (m, n)
    assert out.dtype == (torch.bfloat16 if kind == "fp8" else a.dtype)
    err, bound = (out.double() - want).abs(), off + OUT_HALF[out.dtype] * (want.abs() + off)
    assert (err <= bound).all(), f"off by {(err / bound).max()} of the bound"


@gpu
@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh"])
@pytest.mark.parametrize("kind", ["bf16", "fp16", "fp8"])
@pytest.mark.parametrize("m, n, k", [(1, 1, 32), (1, 96, 4096), (17, 33, 1056), (48, 64, 512),
                                     (130, 301, 544), (513, 256, 288)])
def test_gated(m, n, k, kind, act):
    import flashinfer_amd as fi

    torch.manual_seed(m * n + k)
    a, a_scale, a64 = activations(m, k, kind)
    b, b_scale = weights4(2 * n, k)
    w64 = from4(b, b_scale)
    g, u = a64 @ w64[:n].T, a64 @ w64[n:].T
    og, ou = product_off(a64, w64[:n], kind), product_off(a64, w64[n:], kind)
    want = act64(g, act) * u
    # |act'| <= 1.13; the activation itself is off by a few roundings of g
    og = 1.13 * og + 8 * 2.0 ** -24 * g.abs()
    off = og * (u.abs() + ou) + act64(g, act).abs() * ou
    for dtype in (torch.bfloat16, torch.float16):
        out = fi.gemm_mxfp4_nt_gated(a, b, b_scale, a_scale, activation=act, out_dtype=dtype)
        assert out.shape == (m, n) and out.dtype == dtype
        err = (out.double() - want).abs()
        # fp16 has a least step of 2^-24
        bound = off + OUT_HALF[dtype] * (want.abs() + off) + 2.0 ** -25
        assert (err <= bound).all(), f"off by {(err / bound).max()} of the bound"
    if n % BLOCK == 0:
        q, s = fi.gemm_mxfp4_nt_gated(a, b, b_scale, a_scale, activation=act, out_dtype=FP8)
        assert q.shape == (m, n) and s.shape == (m, n // BLOCK)
        check8(q, s, want, off)


@gpu
@pytest.mark.parametrize("m", [12, 20, 50, 90])
@pytest.mark.parametrize("kind", ["bf16", "fp16", "fp8"])
def test_every_scale_and_special_values(kind, m):
    """Scales from the least to the largest that keep the result finite, NaN
    scales, and NaN and infinite activations."""
    import flashinfer_amd as fi

    torch.manual_seed(0)
    n, k = 200, 256
    a, a_scale, a64 = activations(m, k, kind)
    b, _ = weights4(n, k)
    b_scale = torch.arange(n, device="cuda").to(torch.uint8).unsqueeze(1).repeat(1, k // BLOCK)
    b_scale[:, 1] = 120  # beside blocks of an ordinary size
    w64 = from4(b, b_scale)
    want, off = a64 @ w64.T, product_off(a64, w64, kind)
    out = fi.gemm_mxfp4_nt(a, b, b_scale, a_scale, out_dtype=torch.bfloat16)
    err, bound = (out.double() - want).abs(), off + OUT_HALF[out.dtype] * (want.abs() + off)
    assert (err <= bound).all(), f"off by {(err / bound).max()} of the bound"

    b_scale[:] = 120
    w64 = from4(b, b_scale)
    clean = fi.gemm_mxfp4_nt(a, b, b_scale, a_scale)
    b_scale[5, 3] = 255
    out = fi.gemm_mxfp4_nt(a, b, b_scale, a_scale)
    assert out[:, 5].isnan().all()
    out[:, 5] = clean[:, 5]
    if kind == "fp16":
        # the NaN scale takes its tile to the split of a: the same sums in
        # another order, and two roundings
        off = 2 * product_off(a64, w64, kind) + 2 * OUT_HALF[out.dtype] * clean.double().abs()
        assert ((out.double() - clean.double()).abs() <= off).all()
    else:
        assert torch.equal(out, clean), "a NaN weight reached another output"
    b_scale[5, 3] = 120
    if kind == "fp8":
        a_scale[7, 2] = 255
    else:
        a[7, 70] = math.nan
        a[8, 70] = math.inf
    out = fi.gemm_mxfp4_nt(a, b, b_scale, a_scale)
    assert out[7].isnan().all()
    if kind != "fp8":
        w = w64[:, 70]
        assert out[8, w == 0].isnan().all()
        assert torch.equal(out[8, w != 0].double(), torch.sign(w[w != 0]) * math.inf)
        out[8] = clean[8]
    out[7] = clean[7]
    assert torch.equal(out, clean), "a NaN row reached another output"


@gpu
@pytest.mark.parametrize("kind", ["bf16", "fp16", "fp8"])
@pytest.mark.parametrize("m, n, k", [(24, 12512, 64), (20, 64, 9248), (40, 160, 8480), (200, 1568, 288),
                                     (33, 10272, 160), (100, 10528, 96), (520, 4256, 96),
                                     (1300, 6528, 608), (1, 64, 12320), (16, 32, 6176), (5, 12320, 160),
                                     (3, 16512, 96), (8, 32, 6176), (20, 2592, 6176), (24, 4128, 416),
                                     (32, 8224, 96), (64, 2080, 6240), (50, 8224, 96), (48, 608, 96), (24, 1056, 6176),
                                     (100, 4192, 96), (70, 4224, 96)] + EVERY_GATED)
def test_gated_tiles(m, n, k, kind):
    import flashinfer_amd as fi

    torch.manual_seed(m * n + k)
    a, a_scale, a64 = activations(m, k, kind)
    b, b_scale = weights4(2 * n, k)
    w64 = from4(b, b_scale)
    g, u = a64 @ w64[:n].T, a64 @ w64[n:].T
    og, ou = product_off(a64, w64[:n], kind), product_off(a64, w64[n:], kind)
    want = act64(g, "silu") * u
    og = 1.13 * og + 8 * 2.0 ** -24 * g.abs()
    off = og * (u.abs() + ou) + act64(g, "silu").abs() * ou
    out = fi.gemm_mxfp4_nt_gated(a, b, b_scale, a_scale, out_dtype=torch.bfloat16)
    err, bound = (out.double() - want).abs(), off + 2.0 ** -8 * (want.abs() + off)
    assert (err <= bound).all(), f"off by {(err / bound).max()} of the bound"
    q, s = fi.gemm_mxfp4_nt_gated(a, b, b_scale, a_scale, out_dtype=FP8)
    check8(q, s, want, off)


@gpu
@pytest.mark.parametrize("m, n, k", [(3, 40, 160), (24, 12500, 64), (40, 300, 8480), (200, 3100, 288),
                                     (32, 5000, 416), (60, 5000, 416), (70, 8200, 96), (100, 8200, 96),
                                     (100, 10500, 96), (520, 8450, 96), (1300, 13002, 96)])
def test_fp16_with_weights_outside_its_range(m, n, k):
    """Blocks whose weights fp16 does not hold, some of a tile and some tiles:
    the results are as exact as elsewhere, and the other tiles' too."""
    import flashinfer_amd as fi

    torch.manual_seed(m)
    a, _, a64 = activations(m, k, "fp16")
    b, b_scale = weights4(n, k)
    b_scale[n // 3, 0], b_scale[n // 3, -1] = 103, 98  # below 2^-23, and far below
    b_scale[-1, -1] = 141                              # 6 * 2^14 is no fp16
    a[m // 2, :32] = 0
    a64 = a.double()
    w64 = from4(b, b_scale)
    want, off = a64 @ w64.T, product_off(a64, w64, "fp16")
    out = fi.gemm_mxfp4_nt(a, b, b_scale, out_dtype=torch.bfloat16)
    err, bound = (out.double() - want).abs(), off + 2.0 ** -8 * (want.abs() + off)
    assert (err <= bound).all(), f"off by {(err / bound).max()} of the bound"


@gpu
@pytest.mark.parametrize("kind", ["bf16", "fp16", "fp8"])
@pytest.mark.parametrize("m, n, k", [(1, 70, 6176), (40, 300, 8480), (100, 600, 1056), (300, 3100, 288),
                                     (30, 5000, 6176), (60, 5000, 416)])
def test_results_repeat_bit_by_bit(m, n, k, kind):
    """Sums are joined in a fixed order, by waves, by parts of a workgroup and
    by workgroups; two streams at once share nothing."""
    import flashinfer_amd as fi

    torch.manual_seed(0)
    a, a_scale, _ = activations(m, k, kind)
    b, b_scale = weights4(n, k)
    want = fi.gemm_mxfp4_nt(a, b, b_scale, a_scale)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for i in range(6):
        with torch.cuda.stream(streams[i % 2]):
            outs.append(fi.gemm_mxfp4_nt(a, b, b_scale, a_scale))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = fi.gemm_mxfp4_nt(a, b, b_scale, a_scale)
    for _ in range(3):
        out.zero_()
        g.replay()
        eager = fi.gemm_mxfp4_nt(a, b, b_scale, a_scale)
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(eager, want)


@gpu
@pytest.mark.parametrize("m", [40, 70])
def test_rows_too_far_apart_for_32_bits(m):
    """A tile counts bytes in 32 bits; rows 16 MB apart do not fit it."""
    import flashinfer_amd as fi

    torch.manual_seed(0)
    n, k = 96, 256
    wide = torch.zeros(m, (1 << 23) + 8, dtype=torch.bfloat16, device="cuda")
    wide[:, :k] = torch.randn(m, k, device="cuda")
    b, b_scale = weights4(n, k)
    want = fi.gemm_mxfp4_nt(wide[:, :k].contiguous(), b, b_scale)
    got = fi.gemm_mxfp4_nt(wide[:, :k], b, b_scale)
    torch.testing.assert_close(got, want, rtol=2.0 ** -7, atol=1e-3)


@gpu
def test_more_rows_than_one_launch():
    """2^26 workgroups of 64 lanes would be one thread more than a launch takes."""
    import flashinfer_amd as fi

    rows = 2 ** 26 + 3
    row = torch.arange(1, 33, device="cuda", dtype=torch.bfloat16)
    x = row * (torch.arange(rows, device="cuda") % 2 + 1).to(torch.bfloat16)[:, None]
    w = torch.ones(32, device="cuda", dtype=torch.bfloat16)
    for f in (lambda t: fi.mxfp8_quantize(t), lambda t: fi.rmsnorm_mxfp8_quant(t, w)):
        q, s = f(x)
        want_q, want_s = f(x[:2])
        for i in range(2):
            assert bool((q[i::2].view(torch.uint8) == want_q[i].view(torch.uint8)).all())
            assert bool((s[i::2] == want_s[i]).all())


@gpu
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("m, n", [(33000, 65600), (16, 2 ** 25)])
def test_outputs_past_31_bits(m, n, gated):
    """More than 2^31 outputs, or bytes of them: every row of the last columns."""
    import flashinfer_amd as fi

    torch.manual_seed(0)
    k = 32
    a = torch.randn(m, k, device="cuda").to(torch.bfloat16)
    b, b_scale = weights4(64, k)
    few = (b, b_scale)
    rows = 2 * n if gated else n
    b = torch.zeros(rows, k // 2, dtype=torch.uint8, device="cuda")
    b_scale = torch.full((rows, k // 32), 127, dtype=torch.uint8, device="cuda")
    for at, of in ((n - 32, 0), (rows - 32, 32)) if gated else ((n - 64, 0), (n - 32, 32)):
        b[at:at + 32], b_scale[at:at + 32] = few[0][of:of + 32], few[1][of:of + 32]
    if gated:
        got = fi.gemm_mxfp4_nt_gated(a, b, b_scale, out_dtype=FP8)
        want = fi.gemm_mxfp4_nt_gated(a, *few, out_dtype=FP8)
        assert torch.equal(got[1][:, -1], want[1][:, 0])
        assert torch.equal(got[0][:, -32:].view(torch.uint8), want[0].view(torch.uint8))
        assert not got[0][:, :32].view(torch.uint8).any()
    else:
        got, want = fi.gemm_mxfp4_nt(a, b, b_scale), fi.gemm_mxfp4_nt(a, *few)
        assert torch.equal(got[:, -64:], want)
        assert not got[:, :64].any()


@gpu
@pytest.mark.parametrize("kind", ["bf16", "fp16", "fp8"])
@pytest.mark.parametrize("m", [1, 16, 24, 40, 300])
def test_rows_apart_and_outputs_given(m, kind):
    """Strided rows of a, an output inside a wider tensor, and nothing written
    beside it; NaN lies where nothing may be read."""
    import flashinfer_amd as fi

    torch.manual_seed(m)
    n, k = 77, 96
    a, a_scale, a64 = activations(m, k, kind)
    b, b_scale = weights4(n, k)
    wide = torch.full((m, 2 * k), math.nan, device="cuda").to(a.dtype)
    wide[:, :k] = a
    want = fi.gemm_mxfp4_nt(a, b, b_scale, a_scale)
    box = torch.full((m + 2, n + 5), 7.0, dtype=want.dtype, device="cuda")
    got = fi.gemm_mxfp4_nt(wide[:, :k], b, b_scale, a_scale, out=box[1:-1, 2:2 + n])
    assert got.data_ptr() == box[1:, 2:].data_ptr()
    assert torch.equal(got, want)
    box[1:-1, 2:2 + n] = 7.0
    assert (box == 7.0).all(), "something beside the output was written"
    b, b_scale = weights4(128, k)
    want, want_s = fi.gemm_mxfp4_nt_gated(a, b, b_scale, a_scale, out_dtype=FP8)
    box = torch.full((m + 2, 80), 7, dtype=torch.uint8, device="cuda")
    out_s = torch.zeros_like(want_s)
    q, s = fi.gemm_mxfp4_nt_gated(wide[:, :k], b, b_scale, a_scale,
                                  out=box.view(FP8)[1:-1, 8:72], out_scale=out_s)
    assert s.data_ptr() == out_s.data_ptr() and torch.equal(out_s, want_s)
    assert torch.equal(q.view(torch.uint8), want.view(torch.uint8))
    box[1:-1, 8:72] = 7
    assert (box == 7).all(), "something beside the output was written"


@gpu
def test_empty_products():
    import flashinfer_amd as fi

    a, _, _ = activations(4, 64, "bf16")
    b, s = weights4(8, 64)
    assert fi.gemm_mxfp4_nt(a[:0], b, s).shape == (0, 8)
    assert fi.gemm_mxfp4_nt(a, b[:0], s[:0]).shape == (4, 0)
    q, qs = fi.gemm_mxfp4_nt_gated(a[:0], *weights4(64, 64), out_dtype=FP8)
    assert q.shape == (0, 32) and qs.shape == (0, 1)


# ------------------------------------------------------------ a layer's second half

class Block:
    def __init__(self, hidden, inter):
        torch.manual_seed(1)
        self.norm = (1 + 0.2 * torch.randn(hidden, device="cuda")).bfloat16()
        self.w13 = weights4(2 * inter, hidden, spread=1)
        self.w2 = weights4(hidden, inter, spread=1)

    def __call__(self, x, residual):
        import flashinfer_amd as fi

        a, s = fi.fused_add_rmsnorm_mxfp8_quant(x, residual, self.norm)
        h, hs = fi.gemm_mxfp4_nt_gated(a, *self.w13, s, out_dtype=FP8)
        return fi.gemm_mxfp4_nt(h, *self.w2, hs)


@gpu
@pytest.mark.parametrize("m", [1, 5, 64, 200])
def test_block_follows_its_definition(m):
    """The residual's addition, the norm, the gated block and the down
    projection in a run. Each step is held to the definition on the 8-bit
    values that the step before it wrote."""
    import flashinfer_amd as fi

    hidden, inter = 512, 1408
    block = Block(hidden, inter)
    x = torch.randn(m, hidden, device="cuda").bfloat16()
    r = torch.randn(m, hidden, device="cuda").bfloat16()
    r1 = r.clone()
    out = block(x, r1)
    want_r = (x.float() + r.float()).bfloat16()
    assert torch.equal(r1, want_r)
    a, s = fi.rmsnorm_mxfp8_quant(want_r, block.norm)
    y = norm64(want_r, block.norm, 1e-6)
    check8(a, s, y, norm_off(y, hidden))
    a64, w = from8(a, s), from4(*block.w13)
    g, u = a64 @ w[:inter].T, a64 @ w[inter:].T
    h64 = act64(g, "silu") * u
    h, hs = fi.gemm_mxfp4_nt_gated(a, *block.w13, s, out_dtype=FP8)
    og = 1.13 * product_off(a64, w[:inter], "fp8") + 2.0 ** -21 * g.abs()
    ou = product_off(a64, w[inter:], "fp8")
    check8(h, hs, h64, og * (u.abs() + ou) + act64(g, "silu").abs() * ou)
    h64, w2 = from8(h, hs), from4(*block.w2)
    want, off = h64 @ w2.T, product_off(h64, w2, "fp8")
    assert ((out.double() - want).abs() <= off + 2.0 ** -8 * (want.abs() + off)).all()


@gpu
@pytest.mark.parametrize("m", [1, 40, 300])
def test_block_in_a_graph_and_on_another_stream(m):
    """Two captured graphs of unlike inputs, replayed in turn with eager runs
    between them, give the eager results bit by bit every time."""
    hidden, inter = 512, 1408
    block = Block(hidden, inter)
    xs = [torch.randn(m, hidden, device="cuda").bfloat16() for _ in range(2)]
    rs = [torch.randn(m, hidden, device="cuda").bfloat16() for _ in range(2)]
    want = [block(x, r.clone()) for x, r in zip(xs, rs)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [block(x, r.clone()) for x, r in zip(xs, rs)]
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graphs, outs, held = [], [], []
    for x, r in zip(xs, rs):
        work = r.clone()
        with torch.cuda.stream(side):
            block(x, work)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(block(x, work))
        graphs.append(g)
        held.append(work)
    for _ in range(3):
        for i in (0, 1, 1, 0):
            held[i].copy_(rs[i])
            graphs[i].replay()
            eager = block(xs[1 - i], rs[1 - i].clone())
            torch.cuda.synchronize()
            assert torch.equal(outs[i], want[i])
            assert torch.equal(eager, want[1 - i])
