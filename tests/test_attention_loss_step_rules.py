"""Rules that the kernels of attention, the loss from hidden rows and the optimiser's step keep, read off their sources: every wait has a limit, whoever waits leaves in order."""
import re
from pathlib import Path

import pytest

CUDA = Path(__file__).resolve().parent.parent / "csrc" / "cuda"
SOURCES = ["hc_attention.cu", "hc_loss.cu", "hc_adamw.cu", "hc_tensor.cuh"]


def _code(name):
    return re.sub(r"//[^\n]*", "", (CUDA / name).read_text())


def _body(code, start):
    at = code.index(start)
    depth, i = 0, code.index("{", at)
    for i in range(i, len(code)):
        depth += {"{": 1, "}": -1}.get(code[i], 0)
        if depth == 0:
            return code[at:i + 1]


def _without_lambdas(code):
    while (at := re.search(r"\[&?\](\([^{;]*\))? \{", code)):
        code = code[:at.start()] + code[at.start() + len(_body(code[at.start():], code[at.start():at.end()])):]
    return code


@pytest.mark.parametrize("name", SOURCES)
def test_waits_have_a_limit(name):
    code = _code(name)
    if name == "hc_attention.cu":
        wait = _body(code, "bool attn_wait(")
        assert "kAttnLimitNs" in wait and "gave_up" in wait and "return false" in wait
        code = code.replace(wait, "")
        assert all("kAttnLimitNs" in call for call in re.findall(r"mbar_wait_bounded\(([^;]*);", code))
    assert not re.search(r"mbarrier\.(try_wait|test_wait)|mbar_try_wait|mbar_wait\(", code)
    assert not re.search(r"ld\.(acquire|volatile|relaxed)\.|atomicCAS|while \(\s*(true|1|!)", code)
    assert '"bar.sync' not in code


def test_clusters_meet_outside_of_the_roles():
    """A cluster's barrier has no limit: all threads of all CTAs come to it in any case, behind the barrier of the whole CTA that every role ends at."""
    code = _code("hc_attention.cu")
    assert len(re.findall(r"barrier\.cluster", code)) == 2  # arrive and wait, in one place
    for kernel in ("hc_attention_kernel(", "hc_attention_backward_kernel("):
        body = _body(code[code.index("__global__ void __launch_bounds__(AttnShape<kD>::k" + ("Forward" if kernel == "hc_attention_kernel(" else "Backward")):], kernel)
        ended = body.split("attn_end<S::kColumns>(tmem);")
        assert len(ended) == 2 and "cluster_meet" not in ended[0] and ended[1].count("cluster_meet(p.splits);") == 2
        assert "return;" not in _without_lambdas(ended[0].split("attn_begin<")[1])
    few = _without_lambdas(_body(code, "hc_attention_few_kernel("))
    assert re.findall(r"[^;{}]*return;", few) == ["\n  if (p.splits == 1) return;"] and few.count("cluster_meet(p.splits);") == 2


def test_kernels_that_begin_beside_the_one_before_them():
    """They wait for its results (griddepcontrol.wait) before they read them, and nothing lets loads of these go through the cache that may hold what was there before."""
    for name, kernels in (("hc_attention.cu", ["hc_attention_backward_kernel"]), ("hc_loss.cu", ["hc_loss_join_row_kernel"])):
        code = _code(name)
        beside = re.findall(r"launch_with\((?:dev::)?(\w+)[^;]*, true, ", code)
        beside += re.findall(r"launch_with\((?:dev::)?(\w+)[^;]*, most != nullptr, ", code)
        assert set(beside) == set(kernels)
        for kernel in kernels:
            text = _body(code, kernel + "(")
            assert "__restrict__" not in text and "__ldg" not in code and "grid_dependency_wait();" in text
    join = _body(_code("hc_loss.cu"), "hc_loss_join_row_kernel(")
    assert "[" not in join.split("grid_dependency_wait();")[0].split("tops[32], totals[32];")[1].replace("[](", "")
    keys = _body(_code("hc_attention.cu"), "hc_attention_backward_kernel(")
    assert keys.index("if (kKeys && lane == 0) grid_dependency_wait();") < keys.index("p.delta + side")
    assert keys.index("if (kF16) grid_dependency_wait();") < keys.index("ds_power(p.most")


def test_no_load_goes_to_several_ctas():
    assert "multicast" not in _code("hc_attention.cu") and "multicast" not in _code("hc_loss.cu")


def test_no_other_sums_are_added_to_by_atomics():
    """Atomics find the largest of something, which has no order, and set the status."""
    for name in SOURCES:
        assert set(re.findall(r"atomic\w+", _code(name))) <= {"atomicMax"}
