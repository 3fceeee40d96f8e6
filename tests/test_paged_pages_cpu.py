"""The paged cache hands its pages out once each, and takes them back from the sequence that is named."""
import random

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


def test_no_page_is_held_twice():
    """Random reserves and releases: every page is free or held by one sequence, the table names just those held,
    and a sequence keeps the pages it had."""
    rng = random.Random(3)
    c = _cache(pages=9, seqs=4, max_tokens=80)
    want = [[] for _ in range(4)]
    refused = 0
    for _ in range(600):
        seq = rng.randrange(4)
        if rng.random() < 0.3:
            c.release(seq)
            want[seq] = []
        else:
            tokens = rng.randint(0, 80)
            need = -(-tokens // 16) - len(want[seq])
            if need > 9 - sum(map(len, want)):
                with pytest.raises(RuntimeError, match="full"):
                    c.reserve(seq, tokens)
                refused += 1
            else:
                c.reserve(seq, tokens)
                got = _held(c)[seq]
                assert got[:len(want[seq])] == want[seq] and len(got) == len(want[seq]) + max(0, need)
                want[seq] = got
        held = [p for row in _held(c) for p in row]
        assert _held(c) == want and len(set(held)) == len(held) and all(0 <= p < 9 for p in held)
        assert c.free_pages() == 9 - len(held)
    assert refused > 20
