"""Host logic of the paged cache and the rotary tables, and the C entry points' refusals (nothing is launched)."""
import ctypes
import math

import pytest
import torch


@pytest.fixture(scope="module")
def lib():
    from epure import _native
    return _native.load_library()


def test_frequencies():
    from epure.rotary import rope_frequencies
    base, gain = rope_frequencies(64, theta=1e4)
    assert gain == 1.0 and float(base[0]) == 1.0 and math.isclose(float(base[-1]), 1e4 ** (-62 / 64))
    lin, _ = rope_frequencies(64, theta=1e4, scaling="linear", factor=4.0)
    assert torch.allclose(lin * 4, base, rtol=1e-15)
    ntk, _ = rope_frequencies(64, theta=1e4, scaling="ntk", factor=4.0)
    assert float(ntk[0]) == 1.0 and math.isclose(float(ntk[-1]) * 4, float(base[-1]), rel_tol=1e-12)
    bands, _ = rope_frequencies(128, theta=5e5, scaling="bands", factor=8.0, original_max=8192)
    ref, _ = rope_frequencies(128, theta=5e5)
    wave = 2 * math.pi / ref
    assert torch.equal(bands[wave < 8192 / 4], ref[wave < 8192 / 4])
    assert torch.allclose(bands[wave > 8192] * 8, ref[wave > 8192], rtol=1e-15)
    assert bool((bands <= ref).all()) and bool((bands >= ref / 8 * (1 - 1e-12)).all())
    yarn, gain = rope_frequencies(128, theta=1e4, scaling="yarn", factor=16.0, original_max=4096)
    ref, _ = rope_frequencies(128, theta=1e4)
    assert math.isclose(gain, 0.1 * math.log(16.0) + 1)
    assert float(yarn[0]) == float(ref[0]) and math.isclose(float(yarn[-1]) * 16, float(ref[-1]), rel_tol=1e-12)
    for bad in (dict(rotary_dim=7), dict(rotary_dim=0), dict(rotary_dim=8, scaling="x"),
                dict(rotary_dim=8, factor=0.0, scaling="linear"), dict(rotary_dim=8, scaling="bands", low=4.0, high=4.0)):
        with pytest.raises(ValueError):
            rope_frequencies(**bad)


def test_tables_keep_precision_at_long_positions():
    """Angles in 64 bits: float32 tables are right to their own rounding at position 131071."""
    from epure.rotary import rope_tables
    cos, sin = rope_tables(8, 131072, "cpu", theta=1e4)
    a = 131071.0 * 1e4 ** (-2 / 8)
    assert abs(float(cos[131071, 1]) - math.cos(a)) <= 2.0 ** -24 and abs(float(sin[131071, 1]) - math.sin(a)) <= 2.0 ** -24


def test_cache_hands_pages_out():
    from epure.paged import PagedKVCache
    c = PagedKVCache(2, 6, 16, 2, 32, seqs=3, max_tokens=64, device="cpu", format="int8")
    assert c.k.shape == (2, 6, 2, 16, 32) and c.k.dtype == torch.int8 and c.table.shape == (3, 4)
    c.reserve(0, 17)
    c.reserve(1, 1)
    c.reserve(0, 20)                                   # already there
    assert c.free_pages() == 3 and c.table[0, :2].tolist() == [0, 1] and c.table[1, 0] == 2
    c.reserve(0, 33)
    assert c.table[0].tolist() == [0, 1, 3, -1]
    with pytest.raises(RuntimeError, match="full"):
        c.reserve(2, 64)
    assert c.free_pages() == 2                         # nothing taken by the refused call
    c.release(0)
    assert c.free_pages() == 5 and c.table[0].tolist() == [-1] * 4
    c.reserve(2, 64)
    assert sorted(c.table[2].tolist() + c.table[1, :1].tolist()) == [0, 1, 2, 3, 4] or c.free_pages() == 1
    with pytest.raises(ValueError, match="max_tokens"):
        c.reserve(1, 65)
    with pytest.raises(IndexError):
        c.reserve(3, 1)
    p = c.layer(1)
    assert p.k.data_ptr() == c.k[1].data_ptr() and p.k_scale.shape == (6, 2, 16)
    assert PagedKVCache(1, 2, 16, 2, 32, 1, 32, device="cpu").layer(0).k_scale is None
    for bad in (dict(format="int4"), dict(head_dim=20), dict(pages=0)):
        kw = dict(layers=1, pages=2, page_size=16, kv_heads=2, head_dim=32, seqs=1, max_tokens=32, device="cpu")
        with pytest.raises(ValueError):
            PagedKVCache(**{**kw, **bad})


def _pages(**kw):
    from epure._native import EpqPages
    p = EpqPages()
    p.k = p.v = p.table = 4096                         # never dereferenced: validation fails first
    p.page_stride, p.table_stride, p.pages = 2 * 16 * 64, 4, 8
    p.seqs, p.max_pages, p.page_size, p.kv_heads, p.head_dim, p.format = 2, 4, 16, 2, 64, 0
    for k, v in kw.items():
        setattr(p, k, v)
    return p


def _heads(heads=2, **kw):
    from epure._native import EpqHeads
    h = EpqHeads(4096, heads * 64, 64, heads, 0)
    for k, v in kw.items():
        setattr(h, k, v)
    return h


BAD_PAGES = [("k", None, -1), ("kv_heads", 0, -1), ("page_size", 0, -1), ("pages", 0, -1), ("head_dim", 24, -8),
             ("head_dim", 512, -8), ("format", 3, -1), ("format", 1, -1), ("page_stride", 64, -2),
             ("table_stride", 3, -2), ("k", 4104, -4), ("max_pages", 2 ** 28, -8), ("table", None, -1),
             ("kv_heads", 70000, -8)]


@pytest.mark.parametrize("field,value,code", BAD_PAGES)
def test_bad_pages_rejected(lib, field, value, code):
    p = _pages(**{field: value})
    P = ctypes.c_void_p(4096)
    h = _heads()
    assert lib.epq_paged_read(ctypes.byref(p), P, P, 1, P, P, 2, None) == code
    assert lib.epq_paged_write(ctypes.byref(p), None, None, ctypes.byref(h), ctypes.byref(h), P, P, 1, None, None, 0,
                               0, 0, 0, 1e-6, 2, None) == code
    assert lib.epq_paged_attend(ctypes.byref(p), ctypes.byref(_heads(4)), None, P, 1, 1.0, 0, P, None, 2, P, 1 << 30,
                                None) == code
    assert lib.epq_last_error()


def test_bad_calls_rejected(lib):
    from epure._native import EpqHeads
    P = ctypes.c_void_p(4096)
    p, h = _pages(), _heads()
    ref = ctypes.byref

    def attend(q=None, batch=1, window=0, dtype=2, ws=1 << 30, at=4096, pages=p):
        return lib.epq_paged_attend(ref(pages), ref(q or _heads(4)), None, P, batch, 1.0, window, P, None, dtype,
                                    ctypes.c_void_p(at), ws, None)

    assert attend(batch=-1) == -1 and attend(window=-1) == -1
    assert attend(dtype=0) == -3
    assert attend(q=_heads(3)) == -2 and attend(batch=3) == -2
    assert attend(q=_heads(4, data=4098)) == -4 and attend(q=_heads(4, stride_row=255)) == -4
    assert attend(ws=100) == -6 and attend(at=4100) == -6
    assert attend(batch=40000, pages=_pages(seqs=40000)) == -8
    assert attend(batch=0) == 0
    assert lib.epq_paged_attend_workspace_bytes(ref(p), 1, 4) > 65536 * 4

    def write(q=None, qo=None, k=h, m=1, cos=None, sin=None, max_len=8, r=64, dtype=2):
        return lib.epq_paged_write(ref(p), q and ref(q), qo and ref(qo), ref(k), ref(h), P, P, m, cos, sin, max_len, r, 0,
                                   0, 1e-6, dtype, None)

    assert write(q=h) == -1 and write(cos=P) == -1 and write(m=-1) == -1
    assert write(dtype=9) == -3 and write(k=_heads(3)) == -2
    assert write(cos=P, sin=P, r=66) == -8 and write(cos=P, sin=P, r=7) == -8
    q = _heads(4)
    assert write(q=q, qo=q, cos=P, sin=P, r=20) == -8  # in place needs lanes of 8
    assert write(m=0) == 0
    assert lib.epq_paged_read(ref(p), P, P, 1, ctypes.c_void_p(4100), P, 2, None) == -4

    def rope(x, y, n=1, m=1, hd=64, r=64, dtype=2):
        return lib.epq_rope((EpqHeads * n)(*[x] * n), (EpqHeads * n)(*[y] * n), n, P, m, hd, r, P, P, 8, 0, 0, dtype, None)

    assert rope(h, h, n=3) == -1 and rope(h, h, m=-1) == -1
    assert rope(h, _heads(3)) == -2 and rope(h, h, dtype=5) == -3
    assert rope(h, h, r=3) == -8 and rope(h, h, r=66) == -8 and rope(h, h, hd=2000) == -8
    assert rope(h, h, m=0) == 0
