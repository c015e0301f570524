"""The workspace of attention over a cache in 4 bits goes by the page table that the call has."""
import pytest

from mojolearn_b200 import _native


def need(positions, batch=1, new=600, length=1000, heads=8, kv=8, row_type=1, cache=2):
    return _native.lib().b200i_paged_attention_table_workspace_bytes(-1, row_type, cache, batch * new, batch, heads, kv, 128, new, length, 0, positions)


@pytest.mark.parametrize("batch,positions", [(1, 16), (1, 1008), (1, 1024), (1, 65536), (7, 9360), (3, 21840)])
def test_words_have_room_for_the_positions_of_the_table(batch, positions):
    """Keys and values of 2 bytes, 8 heads of 128, and a number for each page."""
    words = batch * positions * 8 * 128 * 4
    assert words <= 256 << 20
    for length in (1, 1000, 1 << 20):
        assert words <= need(positions, batch, length=length) - need(0, batch, length=length) <= words + batch * positions // 4 + 32


@pytest.mark.parametrize("batch,positions", [(1, 65536 + 16), (2, 65536), (64, 4096), (1 << 20, 1 << 20), (1 << 30, (1 << 31) - 1)])
def test_no_room_is_asked_for_where_there_would_be_none(batch, positions):
    """More than 256 MB of words for the whole table: the codes are read as they are, whatever the lengths are said to be."""
    for length in (1, 1000, 1 << 20):
        assert need(positions, batch, new=600 if batch < 1 << 20 else 1024, length=length) == need(0, batch, new=600 if batch < 1 << 20 else 1024, length=length)


@pytest.mark.parametrize("kw", [{"new": 512}, {"row_type": 0}, {"cache": 1}, {"heads": 32, "new": 128}, {"new": 1}])
def test_no_room_for_words_where_they_are_not_made(kw):
    assert need(1024, **kw) == need(0, **kw) == need(1 << 30, **kw)


@pytest.mark.parametrize("length", [1, 256, 257, 9000])
def test_without_a_table_it_is_one_of_max_length_positions(length):
    plain = _native.lib().b200i_paged_attention_workspace_bytes(-1, 1, 2, 600, 1, 8, 8, 128, 600, length, 0)
    assert plain == need(-(-length // 256) * 256, length=length)
