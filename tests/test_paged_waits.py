"""How the paged kernels go on after a bounded wait that ran out, read from the sources: warps that meet at a barrier all take the same way."""
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "mojolearn_b200", "csrc")


def code(name):
    with open(os.path.join(CSRC, name)) as f:
        return re.sub(r"\s+", " ", re.sub(r"//[^\n]*", "", f.read()))


def test_the_warps_of_few_rows_leave_together():
    """Whether a warp has given up is told by the barrier itself: read from memory behind it, a faster warp could have changed the word before a
    slower one saw it, and would meet nobody at the next barrier."""
    text = code("paged_few.cuh")
    assert text.count("if (few_vote(!alive)) break;") == 2 and "bar.red.or.pred" in text
    assert not re.search(r"if \(dead\) (break|return)", text)
