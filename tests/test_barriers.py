"""Warps that meet at a barrier in a loop (reads the kernels' sources: no GPU)."""
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "xeno-rt_b200", "csrc")


def _closing(text, at, pair):
    """The place behind the bracket that closes the one at ``at``."""
    depth = 0
    for i in range(at, len(text)):
        depth += (text[i] == pair[0]) - (text[i] == pair[1])
        if depth == 0:
            return i + 1
    raise AssertionError("no closing bracket")


def _loops_with_a_named_barrier():
    """(file, header, body) of the outermost loops over a block's tiles in which some of its warps meet."""
    for name in sorted(os.listdir(CSRC)):
        if not name.endswith(".cu"):
            continue
        with open(os.path.join(CSRC, name)) as fh:
            text = re.sub(r"//[^\n]*", "", fh.read())
        end = 0
        for m in re.finditer(r"\bfor \(", text):
            if m.start() < end:
                continue  # inside the loop before
            head = _closing(text, m.end() - 1, "()")
            if text[head:].lstrip()[:1] != "{":
                continue
            stop = _closing(text, text.index("{", head), "{}")
            if re.search(r'"bar\.sync [1-9], ', text[head:stop]):
                end = stop
                yield pytest.param(text[m.start():head], text[head:stop], id=f"{name}: {text[m.start():head][:40]}")


@pytest.mark.parametrize("header,body", list(_loops_with_a_named_barrier()))
def test_no_warp_leaves_a_loop_in_which_others_wait_for_it(header, body):
    """After a wait that ran out (which each warp sees for itself) as little as before."""
    assert not re.search(r"\bok\b", header)
    assert not re.search(r"\b(break|return)\b", body)


def test_there_are_such_loops():
    assert {p.id.split(":")[0] for p in _loops_with_a_named_barrier()} >= {"gemm_int8.cu", "gemm_decode_tcgen05.cu"}


def test_the_last_wait_for_copies_has_a_bound_of_its_own():
    """It runs only where the abort flag is raised: a wait that looked at the flag would end with copies still in flight."""
    with open(os.path.join(CSRC, "tcgen05.cuh")) as fh:
        text = fh.read()
    at = text.index("void mbar_wait_copies(")
    function = text[at:_closing(text, text.index("{", at), "{}")]
    assert "COPY_LIMIT" in function and "abort_flag" not in function and "mbar_wait(" not in function
