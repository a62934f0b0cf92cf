"""Instructions that a warp runs as a whole (``.aligned``): where the code before them can split a warp, its lanes come together again first (``__syncwarp``, or an instruction
that does so itself).  Read off the sources; a barrier of a cluster that some lanes miss has no limit."""
import re
from pathlib import Path

import pytest

CUDA = Path(__file__).resolve().parent.parent / "csrc" / "cuda"
TOGETHER = r"__syncwarp\(\);|__syncthreads\(\);|__all_sync\(|__any_sync\(|attn_wait_all\(|__shfl_xor_sync\("


def _code(name):
    return re.sub(r"//[^\n]*", "", (CUDA / name).read_text())


def _body(code, start):
    at = code.index(start)
    depth, i = 0, code.index("{", at)
    for i in range(i, len(code)):
        depth += {"{": 1, "}": -1}.get(code[i], 0)
        if depth == 0:
            return code[at:i + 1]


def _comes_together(code, before, behind):
    """Between a place where a warp splits and the aligned instruction behind it."""
    at = code.index(before)
    return re.search(TOGETHER, code[at + len(before):code.index(behind, at)]) is not None


def test_a_cluster_is_met_by_whole_warps():
    meet = _body(_code("hc_attention.cu"), "void cluster_meet(")
    assert _comes_together(meet, "{", "barrier.cluster.arrive")


@pytest.mark.parametrize("name,before,behind", [
    ("hc_attention.cu", "sum *= factor;", "if (taken)"),  # some rows' references have grown
    ("hc_attention.cu", "p.delta[side] = delta + lack;", "tc_load32("),  # rows behind the last
])
def test_tensor_memory_is_read_by_whole_warps(name, before, behind):
    assert _comes_together(_code(name), before, behind)


def test_each_piece_of_the_loss_gradient_begins_with_whole_warps():
    """The token's column is one row's affair: the piece behind it is read by the warp as a whole again."""
    grad = _code("hc_gemm.cu").split("if constexpr (kLossGrad")[-1].split("if constexpr (MODE == kGemmLossGrad")[-1].split("const auto piece")[0]
    loop = grad[grad.index("for (int h = 0;"):]
    assert re.search(TOGETHER, loop[:loop.index("tc_load32(")])
