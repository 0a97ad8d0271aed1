"""tcgen05.st is asynchronous: what a kernel stores into TMEM is waited for and fenced
before a barrier tells another warp of it.  Read from the sources, since a kernel that
forgets it gives right results most of the time."""
import glob
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "reflex_b200", "csrc")
SOURCES = sorted(p for p in glob.glob(os.path.join(CSRC, "*.cu")) if "tmem_st16(" in open(p).read())


def forgotten(text):
    """Lines of TMEM stores from which an mbarrier arrival is reached without
    tmem_wait_st() and then tc_fence_before() on the way, in the order of the text."""
    text = re.sub(r"//[^\n]*", "", text)
    step = {"tmem_st16": "stored", "tmem_wait_st": "waited", "tc_fence_before": "fenced"}
    state, at, bad = None, 0, []
    for m in re.finditer(r"\b(tmem_st16|tmem_wait_st|tc_fence_before|mbar_arrive\w*)\(", text):
        what = m.group(1)
        if what == "tmem_st16":
            state, at = "stored", text.count("\n", 0, m.start()) + 1
        elif what == "tmem_wait_st" and state == "stored":
            state = "waited"
        elif what == "tc_fence_before" and state == "waited":
            state = None
        elif what not in step and state is not None:
            bad.append(at)
            state = None
    return bad


@pytest.mark.parametrize("path", SOURCES, ids=os.path.basename)
def test_stores_are_done_before_they_are_announced(path):
    assert forgotten(open(path).read()) == []


def test_what_is_looked_for():
    done = "tmem_st16(a, b);\ntmem_wait_st();\ntc_fence_before();\nmbar_arrive(c);\n"
    assert forgotten(done) == []
    assert forgotten(done.replace("tmem_wait_st();", "")) == [1]
    assert forgotten(done.replace("tc_fence_before();", "")) == [1]
    assert forgotten("tc_fence_before();\ntmem_wait_st();\n" + done.replace("tmem_wait_st();\ntc_fence_before();\n", "")) == [3]
    assert len(SOURCES) >= 4
