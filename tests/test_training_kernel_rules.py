"""Rules that the kernels of the training step's operators keep, read off their sources: every wait has a limit."""
import re
from pathlib import Path

import pytest

CUDA = Path(__file__).resolve().parent.parent / "csrc" / "cuda"
SOURCES = ["hc_norm.cu", "hc_logprobs.cu", "hc_gemm.cu", "hc_linear.cu", "hc_orthogonalize.cu", "hc_train.cuh", "hc_gemm.cuh"]


def _code(name):
    return re.sub(r"//[^\n]*", "", (CUDA / name).read_text())


def _body(code, start):
    """A function's text, from `start` to the brace that closes it."""
    at = code.index(start)
    depth, i = 0, code.index("{", at)
    for i in range(i, len(code)):
        depth += {"{": 1, "}": -1}.get(code[i], 0)
        if depth == 0:
            return code[at:i + 1]


@pytest.mark.parametrize("name", SOURCES)
def test_waits_for_barriers_have_a_limit(name):
    code = _code(name)
    allowed = [_body(code, "bool gemm_wait(")] if name == "hc_gemm.cu" else []
    for body in allowed:
        assert "kGemmLimitNs" in body and "gave_up" in body and "return false" in body
        code = code.replace(body, "")
    assert not re.search(r"mbarrier\.(try_wait|test_wait)|mbar_try_wait\(|mbar_wait\(", code)
    for call in re.findall(r"mbar_wait_bounded\(([^;]*);", code):  # each names its limit
        assert "kGemmLimitNs" in call or "2000ull" in call


@pytest.mark.parametrize("name", SOURCES)
def test_waits_for_other_blocks_have_a_limit(name):
    code = _code(name)
    if name == "hc_gemm.cu":
        meet = _body(code, "bool meet(")
        assert "kGemmLimitNs" in meet and meet.count("return false") == 3
        code = code.replace(meet, "")
    assert not re.search(r"ld\.(acquire|volatile|relaxed)|atomicCAS|while \(\s*(true|1|!)", code)


@pytest.mark.parametrize("name", SOURCES)
def test_hardware_barriers_are_met_by_all(name):
    """Named barriers have no limit: they stand only in the sums of a row's team, which every thread of the team comes to for
    every row, also after a wait that ran out.  Barriers of a pair of CTAs: where the kernel begins and ends."""
    code = _code(name)
    named = re.findall(r'"bar\.sync', code)
    if name == "hc_norm.cu":
        sums = _body(code, "float team_sum(") + _body(code, "void team_sum2(")
        assert len(named) == sums.count('"bar.sync') == 2
        for kernel in ("hc_norm_kernel(const", "hc_norm_backward_kernel(const"):
            rows = _body(_body(code, kernel), "for (; q.row < q.rows; q.next())")
            assert "team_sum" in rows and not re.search(r"\breturn\b|\bbreak\b", rows)
    else:
        assert not named
    assert len(re.findall(r"(?<!void )cluster_sync\(\)", code)) == (2 if name == "hc_gemm.cu" else 0)
