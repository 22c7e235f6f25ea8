"""Which launches may be programmatic, read from the sources (no GPU)."""
import pathlib
import re

import pytest

CSRC = pathlib.Path(__file__).resolve().parents[1] / "dreamx-creator_b200" / "csrc"


def _functions(text):
    """(head, body) of every top-level function of a source file in this code's style: the
    body runs from a line that ends in ``{`` to the next line that is ``}`` alone."""
    for m in re.finditer(r"^((?:template|static|__global__|extern)[^;{}]*)\{\n(.*?)^\}", text,
                         re.S | re.M):
        yield m.group(1), m.group(2)


@pytest.mark.parametrize("name,kernels", [
    ("int8_gemm.cu", {"split_kernel", "pair_kernel"}), ("cross_attn.cu", {"token_kernel"})])
def test_clusters_are_never_launched_programmatically(name, kernels):
    """The kernels of these files that run as clusters go through launch_clusters or
    launch_plain, which set no programmatic attribute; SRDIT_LAUNCH may."""
    text = (CSRC / name).read_text()
    found = set()
    for head, body in _functions(text):
        if "__global__" in head and ("__cluster_dims__" in head or "cluster_" in body):
            found.add(re.search(r"(\w+)\(", head.split("__launch_bounds__")[1].split(")", 1)[1])
                      .group(1))
    assert found == kernels
    launches = 0
    for head, body in _functions(text):
        if "__global__" not in head and any(k + "<" in body for k in kernels):
            assert "SRDIT_LAUNCH" not in body, head
            launches += "launch_clusters(" in body or "launch_plain(" in body
    assert launches == len(kernels)


def test_such_launches_have_no_programmatic_attribute():
    text = (CSRC / "srdit_internal.h").read_text()
    for name in ("launch_clusters", "launch_plain"):
        body = re.search(r"^int %s\(.*?^\}" % name, text, re.S | re.M).group(0)
        assert "Programmatic" not in body and "cudaLaunchKernelEx" in body
