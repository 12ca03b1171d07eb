"""What the 8-bit product kernel's source (csrc/f8_mm.cu) has to say for its
waits to order memory, where running it cannot show the difference."""
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "shoehorn_b200", "csrc")


def function(name):
    """The body of a function of f8_mm.cu, comments taken out."""
    src = re.sub(r"//[^\n]*", "", open(os.path.join(CSRC, "f8_mm.cu")).read())
    at = re.search(r"\b%s\([^;{]*\)\s*\{" % name, src)
    depth, i = 1, at.end()
    while depth:
        depth += {"{": 1, "}": -1}.get(src[i], 0)
        i += 1
    return src[at.end():i - 1]


def test_lanes_are_ordered_behind_the_one_that_waited_for_them():
    """A shuffle orders no memory: after one lane's wait the warp has to meet
    in __syncwarp before any lane reads what the barrier hands over."""
    body = function("warp_wait")
    fast, slow = body.split("bar_wait(", 1)
    # the way without it: every lane tested the barrier itself
    assert re.search(r"if \(__all_sync\(~0u, bar_test\(b, parity\)\)\) return true;", fast)
    assert "__shfl_sync" in slow and "__syncwarp()" in slow[slow.index("__shfl_sync"):slow.index("return")]
