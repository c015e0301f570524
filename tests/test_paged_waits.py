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


def test_nothing_is_in_flight_when_a_block_ends():
    """Copies are waited for by the warp that asked for them, also where only the others have given up; products by the thread that issued them,
    before tensor memory is given back. A warp that did not wait for a slot does not give it back, so no barrier is armed twice in a phase."""
    few, many, fine = code("paged_few.cuh"), code("paged_many.cuh"), code("paged_fine.cuh")
    for text in (few, many, fine):
        assert not re.search(r"if \(!alive\)( \{[^}]*)? for \(unsigned i", text)
    for text in (many, fine):
        assert text.count("if (tail_lost) pg_bar_wait(tail, tails & 1u); for (unsigned i = ld > (unsigned)SLOTS ? ld - SLOTS : 0; i < ld; i++) pg_bar_wait(&full[i % SLOTS], (i / SLOTS) & 1u);") == 1
        assert text.count("alive = false, tail_lost = true;") == 1
        assert text.count("if (!alive) { atomicExch(a.c.status, PAGED_WAIT); pg_commit(done); pg_bar_wait(done, 0); }") == 1 and "pg_bar_init(done, 1)" in text
    assert few.count("for (unsigned i = it > (unsigned)SLOTS ? it - SLOTS : 0; i < it; i++) pg_bar_wait(&sm.full[i % SLOTS], (i / SLOTS) & 1u);") == 1
    assert few.count("sent++;") == 2  # the word that there is no more ends a phase of its barrier as an item's queries do
    assert few.count("for (unsigned i = sent > FEW_ITEMS ? sent - FEW_ITEMS : 0; i < sent; i++) pg_bar_wait(") == 1
    assert len(re.findall(r"if \(lane == 0 && alive\) pg_bar_arrive\(&sm\.(?:item_)?empty", few)) == len(re.findall(r"pg_bar_arrive\(&sm\.(?:item_)?empty", few)) == 4
    assert fine.count("if (alive) pg_bar_arrive(stage_empty);") == fine.count("pg_bar_arrive(stage_empty)") == 2
    assert "if (items > 0) pg_bar_wait(stage_full, (items - 1) & 1u);" in fine
