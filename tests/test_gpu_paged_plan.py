"""Paged attention of more units (sequence, key head, up to 16 query heads) than a launch has CTAs: their blocks are
dealt out in runs that go over unit boundaries, and units are cut where the runs end."""
import pytest
import torch
from test_gpu_paged import DEV, _check, _fill, _gen, _gpu, _pages  # noqa: F401 (_gpu: a fixture)

pytestmark = pytest.mark.gpu

MOST_CTAS = 512          # of a launch, whatever the GPU (kMaxGrid)
MIXED = [0, 1, 15, 16, 17, 63, 64, 65, 333, 0, 1000, 500, 0]


def _lengths(units, long=0):
    """MIXED again and again, empty rows between and at both ends, until their units are more than any launch's
    CTAs; then the plan of one piece a CTA cannot hold them."""
    got = []
    while sum(n > 0 for n in got) * units <= MOST_CTAS:
        got += MIXED
    if long:
        got[len(got) // 2] = long
    return got


@pytest.mark.parametrize("fmt,dtype,heads,kv,hd,ps,window,long", [
    ("same", torch.bfloat16, 32, 8, 128, 16, 0, 0), ("same", torch.bfloat16, 32, 8, 128, 16, 100, 0),
    ("same", torch.float16, 8, 8, 64, 48, 0, 20011), ("int8", torch.bfloat16, 32, 8, 128, 64, 0, 20011),
    ("int8", torch.bfloat16, 32, 8, 128, 24, 70, 0), ("fp8", torch.bfloat16, 64, 8, 128, 32, 0, 0),
    ("fp8", torch.float16, 12, 4, 80, 7, 0, 5000), ("same", torch.bfloat16, 12, 4, 80, 16, 0, 0),
    ("int8", torch.float16, 40, 2, 64, 16, 0, 3000), ("same", torch.bfloat16, 24, 2, 256, 5, 0, 2000),
    ("fp8", torch.bfloat16, 4, 4, 256, 16, 300, 0), ("int8", torch.bfloat16, 4, 4, 16, 1, 0, 0)])
def test_more_units_than_ctas(fmt, dtype, heads, kv, hd, ps, window, long):
    from epure import paged
    group = heads // kv
    units = kv * (1 if group <= 8 else -(-group // 16))
    lengths = _lengths(units, long)
    pages = _pages(lengths, kv, hd, ps, fmt, dtype)
    k, v = _fill(pages, lengths, dtype)
    q = (torch.randn(len(lengths), heads, hd, generator=_gen(41), device=DEV) * 2).to(dtype)
    out, lse = _check(pages, q, lengths, k, v, window=window)
    n = torch.tensor(lengths, device=DEV)
    paged.attend(pages, q[:5], n[:5])                  # another plan on the same workspace
    again = paged.attend(pages, q, n, window=window, return_lse=True)
    assert torch.equal(again[0], out) and torch.equal(again[1], lse)


@pytest.mark.parametrize("fmt", ["same", "int8"])
def test_full_batches_of_equal_lengths(fmt):
    """128 sequences of one length: runs end inside units at every distance, and at their ends."""
    for n in (1, 16, 64, 80, 177):
        lengths = [n] * 128
        pages = _pages(lengths, 8, 64, 16, fmt, torch.bfloat16)
        k, v = _fill(pages, lengths, torch.bfloat16)
        q = torch.randn(128, 8, 64, generator=_gen(42), device=DEV).to(torch.bfloat16)
        _check(pages, q, lengths, k, v)


def test_some_sequences_of_many_in_another_order():
    """Rows that name sequences out of order, some twice."""
    from epure import paged
    lengths = _lengths(4)
    pages = _pages(lengths, 4, 128, 16, "int8", torch.bfloat16)
    _fill(pages, lengths, torch.bfloat16)
    q = torch.randn(len(lengths), 16, 128, generator=_gen(43), device=DEV).to(torch.bfloat16)
    n = torch.tensor(lengths, device=DEV)
    want, lse = paged.attend(pages, q, n, return_lse=True)
    pick = torch.randperm(len(lengths), generator=torch.Generator().manual_seed(44)).to(DEV)
    pick = torch.cat((pick, pick[:40]))
    got, got_lse = paged.attend(pages, q[pick], n[pick], seq=pick.int(), return_lse=True)
    # other cuts, so other orders of the same float32 sums: results may round the other way
    assert float((got.float() - want[pick].float()).abs().max()) <= 2.0 ** -7 * float(want.abs().max())
    live = n[pick] > 0
    assert float((got_lse - lse[pick])[live].abs().max()) <= 2.0 ** -18 * float(lse[n > 0].abs().max())
    assert not got[~live].any() and bool(torch.isneginf(got_lse[~live]).all())
