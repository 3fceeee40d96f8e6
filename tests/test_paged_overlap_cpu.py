"""What the rotary and paged C entry points refuse because its rows would be written over one another (no launch)."""
import ctypes
import random

import pytest
from test_paged_cpu import _heads, _pages, lib  # noqa: F401 (lib: a fixture)


def _rope(lib, x, y, m, hd=64):
    from epure._native import EpqHeads
    P = ctypes.c_void_p(4096)
    return lib.epq_rope((EpqHeads * 1)(x), (EpqHeads * 1)(y), 1, P, m, hd, hd, P, P, 8, 0, 0, 2, None)


def _write(lib, q, qo, m):
    P, h, ref = ctypes.c_void_p(4096), _heads(), ctypes.byref
    return lib.epq_paged_write(ref(_pages()), ref(q), ref(qo), ref(h), ref(h), P, P, m, None, None, 0, 0, 0, 0, 1e-6, 2,
                               None)


OVERLAPPING = [(4, 64, 0, 64), (4, 2, 128, 0), (4, 2, 0, 0), (4, 2, 64, 64), (4, 2, 65, 64), (3, 4, 128, 64),
               (2, 8, 100, 150), (4, 2, -64, 64), (4, 2, 128, 32), (5, 7, 450, 100)]


@pytest.mark.parametrize("m,heads,row,head", OVERLAPPING)
def test_outputs_that_overlap_themselves_are_refused(lib, m, heads, row, head):  # noqa: F811
    x = _heads(heads, data=1 << 30)
    y = _heads(heads, stride_row=row, stride_head=head)
    assert _rope(lib, x, y, m) == -2 and b"overlap" in lib.epq_last_error()
    assert _write(lib, x, y, m) == -2 and b"overlap" in lib.epq_last_error()


def test_in_place_with_other_strides_is_refused(lib):  # noqa: F811
    x = _heads(4)
    for y in (_heads(4, stride_row=512), _heads(4, stride_row=64, stride_head=256)):
        assert _rope(lib, x, y, 4) == -2 and _write(lib, x, y, 4) == -2


def test_overlap_rule_matches_the_definition():
    """The rule, restated, against the distances of all pairs of heads (the refusals above run the library's)."""
    def rule(m, H, sr, sh, hd):
        sr, sh = abs(sr), abs(sh)
        if (m > 1 and sr < hd) or (H > 1 and sh < hd):
            return True
        if m <= 1 or H <= 1 or sr // H >= sh or sh // m >= sr:
            return False
        for h in range(1, H):
            r, past = divmod(h * sh, sr)
            if (r < m and past < hd) or (r + 1 < m and sr - past < hd):
                return True
        return False

    rng = random.Random(1)
    seen = [0, 0]
    for _ in range(20000):
        m, H, hd = rng.randint(1, 6), rng.randint(1, 6), rng.randint(2, 8)
        sr, sh = rng.randint(-60, 60), rng.randint(-60, 60)
        at = sorted(r * sr + h * sh for r in range(m) for h in range(H))
        want = any(b - a < hd for a, b in zip(at, at[1:]))
        assert rule(m, H, sr, sh, hd) == want, (m, H, sr, sh, hd)
        seen[want] += 1
    assert min(seen) > 1000
