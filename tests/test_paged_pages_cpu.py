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
