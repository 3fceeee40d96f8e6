"""Refusals of the sparse, shared-prefix and verification entry points, and pages that sequences share (nothing is
launched)."""
import ctypes

import pytest
import torch
from test_paged_cpu import BAD_PAGES, _heads, _pages, lib  # noqa: F401 (lib: a fixture)

P = ctypes.c_void_p(4096)
ref = ctypes.byref


def _bounds(lib, p=None, at=4096, stride=256, dtype=2, batch=1, lengths=P, seq=None):
    return lib.epq_paged_bounds(ref(p or _pages()), ctypes.c_void_p(at), stride, dtype, seq, None, lengths, batch, None)


def _select(lib, p=None, q=None, at=4096, stride=256, kind=2, dtype=2, batch=1, count=4, sinks=1, recent=1, chosen=P, ws=1 << 30,
            work=4096, lengths=P):
    return lib.epq_paged_select(ref(p or _pages()), ctypes.c_void_p(at), stride, kind, ref(q or _heads(4)), dtype, None, lengths, batch,
                                count, sinks, recent, chosen, ctypes.c_void_p(work), ws, None)


def _blocks(lib, p=None, q=None, batch=1, blocks=P, count=4, dtype=2, ws=1 << 30, work=4096):
    return lib.epq_paged_attend_blocks(ref(p or _pages()), ref(q or _heads(4)), None, P, batch, blocks, count, 1.0, P, None, dtype,
                                       ctypes.c_void_p(work), ws, None)


def _shared(lib, p=None, q=None, batch=1, starts=P, prefix=P, groups=1, dtype=2, ws=1 << 34, work=4096, lengths=P):
    return lib.epq_paged_attend_shared(ref(p or _pages()), ref(q or _heads(4)), None, lengths, batch, starts, prefix, groups, 0, 1.0, P,
                                       None, dtype, ctypes.c_void_p(work), ws, None)


@pytest.mark.parametrize("field,value,code", BAD_PAGES)
def test_bad_pages(lib, field, value, code):  # noqa: F811
    p = _pages(**{field: value})
    assert _bounds(lib, p) == code and _select(lib, p) == code and _blocks(lib, p) == code and _shared(lib, p) == code
    assert lib.epq_paged_select_workspace_bytes(ref(p), 1) == code
    assert lib.epq_paged_attend_shared_workspace_bytes(ref(p), 1, 4, 1, 0) == code


def test_bad_bounds_and_selections(lib):  # noqa: F811
    for call in (_bounds, _select):
        assert call(lib, at=0) == -1 and call(lib, at=4104) == -4 and call(lib, stride=260) == -4 and call(lib, stride=248) == -2
        assert call(lib, batch=-1) == -1 and call(lib, batch=3) == -2 and call(lib, lengths=None) == -1 and call(lib, batch=0) == 0
    assert _bounds(lib, dtype=0) == -3 and _bounds(lib, _pages(format=1, k_scale=4096, v_scale=4096, scale_stride=32), dtype=1) == -3
    assert _bounds(lib, batch=70000, seq=P) == -1
    assert _select(lib, kind=0) == -3 and _select(lib, dtype=0) == -3
    assert _select(lib, count=0) == -1 and _select(lib, count=2, sinks=2) == -1 and _select(lib, sinks=-1) == -1
    assert _select(lib, count=2 ** 31 - 1, sinks=2 ** 31 - 1, recent=2 ** 31 - 1) == -1
    assert _select(lib, q=_heads(3)) == -2 and _select(lib, chosen=None) == -1
    assert _select(lib, ws=65536 * 4) == -6 and _select(lib, work=4100) == -6
    assert _select(lib, _pages(seqs=40000), batch=40000) == -8
    assert lib.epq_paged_select_workspace_bytes(ref(_pages()), 2) == 65536 * 4 + 2 * 2 * (4 + 1) * 4        # counters, keys, largest bounds


def test_bad_lists_and_groups(lib):  # noqa: F811
    for call in (_blocks, _shared):
        assert call(lib, batch=-1) == -1 and call(lib, dtype=0) == -3 and call(lib, q=_heads(3)) == -2 and call(lib, batch=3) == -2
        assert call(lib, q=_heads(4, data=4098)) == -4 and call(lib, ws=100) == -6 and call(lib, work=4100) == -6
        assert call(lib, batch=0) == 0 and call(lib, _pages(seqs=40000), batch=40000) == -8
    assert _blocks(lib, count=-1) == -1 and _blocks(lib, blocks=None) == -1
    assert _shared(lib, groups=-1) == -1 and _shared(lib, starts=None) == -1 and _shared(lib, prefix=None) == -1
    assert lib.epq_paged_attend_shared_workspace_bytes(ref(_pages()), 1, 4, -1, 0) == -1


def test_bad_verifications(lib):  # noqa: F811
    from epure._native import EpqProbs

    def verify(p=EpqProbs(4096, 500, 100), q=EpqProbs(4096, 400, 100), x=P, u=P, batch=1, drafts=4, vocab=100, dtype=0, out=P, n=P):
        return lib.epq_verify_drafts(p and ref(p), q and ref(q), x, 4, u, 5, batch, drafts, vocab, dtype, out, n, None)

    assert verify(p=None) == -1 and verify(p=EpqProbs(None, 1, 1)) == -1 and verify(q=EpqProbs(None, 1, 1)) == -1
    assert verify(batch=-1) == -1 and verify(drafts=-1) == -1 and verify(vocab=0) == -1
    assert verify(x=None) == -1 and verify(u=None) == -1 and verify(out=None) == -1 and verify(n=None) == -1
    assert verify(dtype=7) == -3 and verify(p=EpqProbs(4098, 1, 1)) == -4 and verify(q=EpqProbs(4097, 1, 1), dtype=2) == -4
    assert verify(batch=2 ** 29) == -8 and verify(vocab=2 ** 30) == -8
    assert verify(batch=0) == 0


def _cache(**kw):
    from epure.paged import PagedKVCache
    return PagedKVCache(**{**dict(layers=1, pages=6, page_size=16, kv_heads=2, head_dim=32, seqs=3, max_tokens=64, device="cpu"), **kw})


def test_shared_pages_stay_until_their_last_sequence_goes():
    c = _cache()
    c.reserve(0, 40)
    assert c.share(1, 0, 40) == 32 and c.free_pages() == 3
    c.reserve(1, 50)
    assert c.table[1].tolist() == c.table[0, :2].tolist() + [3, 4] and c.free_pages() == 1
    assert c.share(2, 1, 50) == 48                     # a sharer of a sharer
    c.release(0)
    assert c.free_pages() == 2 and c.table[0].tolist() == [-1] * 4
    c.release(1)
    assert c.free_pages() == 3 and c.table[2, :3].tolist() == [0, 1, 3]
    c.reserve(0, 48)                                   # none of the shared ones is handed out
    assert not set(c.table[0, :3].tolist()) & {0, 1, 3}
    c.release(2)
    c.release(0)
    assert c.free_pages() == 6
    c.release(0)
    assert sorted(c._free) == list(range(6)) and not any(c._users)


def test_share_refusals():
    c = _cache()
    c.reserve(0, 20)
    c.reserve(1, 1)
    assert c.share(2, 0, 15) == 0 and c.table[2].tolist() == [-1] * 4
    for bad in ((1, 0, 16), (2, 0, 33), (2, 0, -1)):
        with pytest.raises(ValueError):
            c.share(*bad)
    for bad in ((3, 0, 16), (2, -1, 16)):
        with pytest.raises(IndexError):
            c.share(*bad)
    with pytest.raises(ValueError):
        c.share(0, 0, 16)
    assert c.free_pages() == 3


def test_bounds_of_a_cache():
    assert _cache().bounds is None
    assert _cache(bounds=True).bounds.shape == (1, 6, 2, 2, 32) and _cache(bounds=True).bounds.dtype == torch.bfloat16
    assert _cache(bounds=True, dtype=torch.float16).bounds.dtype == torch.float16
    assert _cache(bounds=True, dtype=torch.float16, format="int8").bounds.dtype == torch.bfloat16
