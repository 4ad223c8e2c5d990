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
