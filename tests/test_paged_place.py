"""Where a call's tables put a sequence (csrc/paged_place.cuh), with the host compiler: whatever they say, its rows lie within the call's
and its positions within the page table's."""
import os
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "mojolearn_b200", "csrc")
PROGRAM = r"""
#include <cstdio>
#include <cstdlib>
#include "paged_place.cuh"
int main(int argc, char **argv) {
    int v[5];
    while (scanf("%d %d %d %d %d", v, v + 1, v + 2, v + 3, v + 4) == 5) {
        const b200i::PagedSeq s = b200i::paged_place(v[0], v[1], v[2], v[3], v[4]);
        printf("%d %d %d %d\n", s.first, s.n, s.length, s.pos0);
    }
}
"""
LOW, HIGH = -(1 << 31), (1 << 31) - 1


@pytest.fixture(scope="module")
def place(tmp_path_factory):
    d = tmp_path_factory.mktemp("place")
    (d / "place.cpp").write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-O1", "-fwrapv", "-I", CSRC, str(d / "place.cpp"), "-o", str(d / "place")], check=True)

    def run(cases):
        text = "".join("%d %d %d %d %d\n" % c for c in cases)
        out = subprocess.run([str(d / "place")], input=text, capture_output=True, text=True, check=True).stdout
        return [tuple(map(int, line.split())) for line in out.splitlines()]
    return run


def test_tables_of_any_words_stay_inside(place):
    odd = [LOW, LOW + 1, -7, -1, 0, 1, 5, 9, 10, 11, 100, HIGH - 1, HIGH]
    cases = [(lo, hi, length, 10, 64) for lo in odd for hi in odd for length in odd]
    for case, (first, n, length, pos0) in zip(cases, place(cases)):
        assert 0 <= first <= 10 and 0 <= n and first + n <= 10, (case, first, n)
        assert 0 <= length <= 64 and pos0 + n <= 64, (case, length, pos0)
        if n:
            assert max(case[0], 0) == first and first + n <= case[1], (case, first, n)


def test_ordinary_tables(place):
    assert place([(0, 3, 20, 10, 64), (3, 10, 64, 10, 64), (5, 5, 7, 10, 64), (2, 9, 3, 10, 64)]) == [(0, 3, 20, 17), (3, 7, 64, 57), (5, 0, 7, 7), (2, 7, 3, -4)]


def test_a_sequence_that_is_not_held_has_no_rows(place):
    """More positions than the table has room for, or offsets that are not the call's: its rows are not moved to other positions."""
    for case in [(0, 3, 65, 10, 64), (0, 3, HIGH, 10, 64), (8, 11, 20, 10, 64), (-1, 3, 20, 10, 64), (5, 2, 20, 10, 64), (LOW, HIGH, 20, 10, 64)]:
        assert place([case])[0][1] == 0, case
    assert place([(0, 3, 64, 10, 64), (4, 4, 65, 10, 64)]) == [(0, 3, 64, 61), (4, 0, 64, 64)]
