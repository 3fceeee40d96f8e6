"""The paged cache hands its pages out once each, and takes them back from the sequence that is named."""
import pytest

from epure.paged import PagedKVCache


def _cache(**kw):
    return PagedKVCache(**{**dict(layers=1, pages=6, page_size=16, kv_heads=2, head_dim=32, seqs=3, max_tokens=64,
                                  device="cpu"), **kw})


def _held(c):
    return [[p for p in row if p >= 0] for row in c.table.tolist()]


def test_release_refuses_sequences_that_are_not():
    c = _cache()
    c.reserve(2, 20)
    held = _held(c)
    for seq in (-1, -3, 3):
        with pytest.raises(IndexError, match="sequence"):
            c.release(seq)
    assert _held(c) == held and c.free_pages() == 4
    c.release(2)
    c.release(2)                                       # nothing held: nothing happens
    assert c.free_pages() == 6 and not any(_held(c))


def test_a_failed_copy_takes_no_pages():
    """The table cannot be written (inside a capture, say): the pages stay free."""
    class Refusing:
        def __setitem__(self, at, value):
            raise RuntimeError("no copy")

    c = _cache()
    c.reserve(0, 17)
    table, c.table = c.table, Refusing()
    with pytest.raises(RuntimeError, match="no copy"):
        c.reserve(0, 64)
    with pytest.raises(RuntimeError, match="no copy"):
        c.reserve(1, 1)
    assert c.free_pages() == 4
    c.table = table
    c.reserve(1, 64)
    assert _held(c) == [[0, 1], [2, 3, 4, 5], []] and c.free_pages() == 0
    c.release(0)
    c.release(1)
    assert c.free_pages() == 6
