"""The kernel that ``ops.linear`` takes for a few rows holds all that it works on in registers, in each of its forms, as the assembler reports them."""
import re
import subprocess

import pytest

from tirocinio_triennale_b200 import _build


@pytest.mark.skipif(_build.nvcc_path() is None, reason="needs nvcc")
def test_few_rows_spill_nothing(tmp_path):
    cuda = _build.CSRC / "cuda"
    flags = [f for f in _build.NVCC_FLAGS if f != "-lineinfo"]
    out = subprocess.run([_build.nvcc_path(), *flags, "-Xptxas", "-v", "-I", str(cuda.parent / "include"), "-cubin", str(cuda / "hc_linear.cu"), "-o", str(tmp_path / "cubin")],
                         capture_output=True, text=True, check=True).stderr
    # results that are stored (of logits, the last parameter's other value, only sums are kept)
    entries = [e for e in out.split("Compiling entry function ")[1:] if re.search(r"hc_few_rows_kernelI\S+Li\dELb[01](ELb0)?EEEv", e.split("'")[1])]
    assert len(entries) == 8
    for e in entries:
        assert re.search(r"(\d+) bytes spill stores, (\d+) bytes spill loads", e).groups() == ("0", "0"), e.split("'")[1]
