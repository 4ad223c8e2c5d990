"""What the MX operators do ahead of a launch, and what their sources promise the
compiler: no GPU is needed for any of it."""
import re
from pathlib import Path

import pytest
import torch

import flashinfer_amd
from flashinfer_amd._lib import has_ext

CSRC = Path(flashinfer_amd.__file__).parent / "csrc"
needs_ext = pytest.mark.skipif(not has_ext(), reason="native extension not built")


def asm_statements():
    for path in sorted([*CSRC.rglob("*.hip"), *CSRC.rglob("*.hpp")]):
        for found in re.finditer(r"\basm\b[^;]*?\((.*?)\);", path.read_text(), re.S):
            yield path.name, found.group(1)


def test_assembly_that_writes_m0_says_so():
    writers = [(name, text) for name, text in asm_statements() if re.search(r"\bs_mov_b32 m0\b", text)]
    assert len(writers) >= 2
    for name, text in writers:
        assert '"m0"' in text.rsplit(":", 1)[-1], f"{name}: {text}"


@needs_ext
@pytest.mark.parametrize("call", [
    lambda fi, x, w: fi.rmsnorm_mxfp8_quant(x, None),
    lambda fi, x, w: fi.fused_add_rmsnorm_mxfp8_quant(x, x.clone(), None),
    lambda fi, x, w: fi.fused_add_rmsnorm_mxfp8_quant(x, None, w),
    lambda fi, x, w: fi.mxfp8_quantize(None),
])
def test_a_missing_operand_is_refused(call):
    """Without its weight a norm would be a quantization, and without its residual
    an addition would be left out."""
    with pytest.raises(TypeError, match="incompatible function arguments"):
        call(flashinfer_amd, torch.zeros(2, 64), torch.zeros(64))


ENTRIES = ["rmsnorm_mxfp8_quant", "fused_add_rmsnorm_mxfp8_quant", "mxfp8_quantize", "mxfp4_quantize",
           "gemm_mxfp4_nt", "gemm_mxfp4_nt_gated"]


@pytest.mark.parametrize("name", ENTRIES)
def test_a_substitute_takes_over_every_entry(name):
    from flashinfer_amd import trace_apply

    trace_apply.enable_apply({name: lambda *args, **kw: (name, args, kw)})
    try:
        assert getattr(flashinfer_amd, name)(1, out=2) == (name, (1,), {"out": 2})
    finally:
        trace_apply.disable_apply()


def test_every_entry_is_logged():
    import os
    import subprocess
    import sys

    code = ("import flashinfer_amd as fi\n"
            f"for name in {ENTRIES}:\n"
            "    try: getattr(fi, name)(None)\n"
            "    except Exception: pass\n")
    run = subprocess.run([sys.executable, "-c", code], env={**os.environ, "FLASHINFER_LOGLEVEL": "1"},
                         cwd=CSRC.parent.parent, capture_output=True, text=True, check=True)
    for name in ENTRIES:
        assert f"[flashinfer_amd] {name}" in run.stderr.splitlines()


def test_mxfp4_quantize_takes_64_bits_as_they_are():
    from test_mx import from4

    w = torch.zeros(4, 32, dtype=torch.float64)
    w[0, :5] = torch.tensor([6, 0.25, 1.25, 2.5, 5], dtype=torch.float64) * (1 + 2.0 ** -40)
    w[0, 0] = 6                   # a step above the middles of two levels: not ties
    w[1, 0] = 6 * (1 + 2.0 ** -40)  # saturates by a little at the scale of 1
    w[2, 0] = 6 * 2.0 ** 127      # no float32, but the largest value of the format
    w[3, 0] = 6 * 2.0 ** 127 * (1 + 2.0 ** -40)
    b, s = flashinfer_amd.mxfp4_quantize(w)
    d = from4(b, s)
    assert torch.equal(d[0, :5], torch.tensor([6, 0.5, 1.5, 3, 6], dtype=torch.float64))
    assert s[1, 0] == 128 and s[2, 0] == 254 and d[2, 0] == w[2, 0]
    assert s[3, 0] == 255 and d[3].isnan().all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32, torch.float64])
def test_mxfp4_quantize_on_the_gpu_is_that_of_the_cpu(dtype):
    gen = torch.Generator().manual_seed(0)
    top = 15 if dtype == torch.float16 else 126
    w = torch.randint(-16, 17, (3, 512, 96), generator=gen).double() / 4  # ties among them
    w += torch.randn(w.shape, generator=gen) * (torch.rand(w.shape, generator=gen) < 0.5)
    w *= torch.exp2(torch.randint(-top - 12, top - 3, (3, 512, 3), generator=gen).double()
                    ).repeat_interleave(32, -1)
    w = w.to(dtype)
    w[0, 0, 3], w[0, 1, 40], w[0, 2] = float("nan"), float("inf"), 0
    b, s = flashinfer_amd.mxfp4_quantize(w)
    got_b, got_s = flashinfer_amd.mxfp4_quantize(w.cuda())
    assert torch.equal(got_s.cpu(), s) and torch.equal(got_b.cpu(), b)
