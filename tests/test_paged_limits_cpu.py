"""Limits of the paged attention's 32-bit counts (no launch)."""
import ctypes

from test_paged_cpu import _heads, _pages, lib  # noqa: F401 (lib: a fixture)


def test_runs_past_32_bits_are_refused(lib):  # noqa: F811
    """2^27 blocks of 16 tokens for each of 8192 key heads: a CTA's share would not fit its 32-bit run."""
    P, ref = ctypes.c_void_p(4096), ctypes.byref

    def attend(heads, max_pages):
        p = _pages(kv_heads=heads, page_size=1024, head_dim=16, max_pages=max_pages, table_stride=max_pages,
                   page_stride=heads * 1024 * 16)
        rc = lib.epq_paged_attend(ref(p), ref(_heads(heads)), None, P, 1, 1.0, 0, P, None, 2, P, 100, None)
        return rc

    assert attend(8192, 2 ** 21 - 1) == -8
    assert b"tokens" in lib.epq_last_error()
    assert attend(8192, 2 ** 17) == -6                 # 2^36 blocks in all are taken (and the workspace is too small)
    assert attend(512, 2 ** 21 - 1) == -6
