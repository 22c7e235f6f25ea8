"""What a kernel does after a wait that ran out, read from the sources (no GPU).

A lane that gave up must not leave the lanes of its warp, nor a warp those that it meets at a
named barrier, to wait for it: those waits have no limit of their own."""
import pathlib
import re

import pytest

CSRC = pathlib.Path(__file__).resolve().parents[1] / "dreamx-creator_b200" / "csrc"
FILES = ("int8_gemm.cu", "cross_attn.cu")


def _code(name):
    return re.sub(r"//[^\n]*", "", (CSRC / name).read_text())


def _without_single_threads(text):
    """The text without the blocks that one thread of a warp runs."""
    out = []
    at = 0
    for m in re.finditer(r"if \([^;{}]*(?:elect_one\(\)|lane == 0|threadIdx\.x == 0)\) \{", text):
        if m.start() < at:
            continue
        depth, end = 1, m.end()
        while depth:
            depth += {"{": 1, "}": -1}.get(text[end], 0)
            end += 1
        out.append(text[at:m.start()])
        at = end
    return "".join(out) + text[at:]


@pytest.mark.parametrize("name", FILES)
def test_a_warp_gives_up_as_one(name):
    """Waits of whole warps have one answer for all lanes, or none is asked for (and the abort
    flag, which ends every later wait, is voted on); only single threads go by their own."""
    text = _code(name)
    assert "mbar_wait" in text
    shared = _without_single_threads(text)
    for m in re.finditer(r"\bmbar_wait\(", shared):
        assert re.search(r"[;{}]\s*$", shared[:m.start()]), shared[m.start() - 40:m.end() + 60]
        call = shared[m.start():shared.index(";", m.end())]
        assert call.endswith("abort_flag)")
        assert "if (__any_sync(0xffffffffu, *abort_flag != 0u)) break;" in shared


@pytest.mark.parametrize("name", FILES)
def test_warps_that_meet_leave_together(name):
    """No warp passes a named barrier that another may have left for good: each says there
    whether it goes on, and all go by the answer."""
    assert "named_barrier_sync" not in _code(name)


def test_the_answer_is_one():
    text = (CSRC / "sm100.cuh").read_text()
    body = re.search(r"bool mbar_wait_warp\(.*?\n\}", text, re.S).group(0)
    assert "__all_sync(0xffffffffu, mbar_wait(" in body
    body = re.search(r"bool named_barrier_all\(.*?\n\}", text, re.S).group(0)
    assert "bar.red.and.pred" in body
