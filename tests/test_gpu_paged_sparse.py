"""Bounds of a cache's pages (paged.summarise), the blocks that they choose (paged.select) and attention over listed
blocks (paged.attend(blocks=))."""
import math
import os
import subprocess
import sys

import pytest
import torch
from conftest import PKG
from test_gpu_paged import DEV, UNIT, _fill, _gen, _gpu, _pages, _tokens  # noqa: F401 (_gpu: a fixture)

pytestmark = pytest.mark.gpu


def _new_bounds(pages, dtype, fill=7.0):
    kind = dtype if pages.k_scale is None else torch.bfloat16
    return torch.full((pages.k.shape[0], pages.k.shape[1], 2, pages.k.shape[3]), fill, dtype=kind, device=DEV)


# -- bounds ------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("fmt", ["same", "int8", "fp8"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("kv,hd,ps", [(8, 128, 64), (2, 64, 16), (3, 80, 7), (1, 256, 1), (4, 16, 48), (2, 48, 24),
                                      (1, 112, 130)])
def test_bounds(fmt, dtype, kv, hd, ps):
    """The least and largest value of the tokens below a row's length, exactly (8-bit: of code * scale, rounded to
    bf16); pages without a new token and slots behind the length are not looked at (they hold NaN)."""
    from epure import paged
    lengths, first = [0, 1, 16, 65, 333, 200, 64, 130], [0, 0, 15, 3, 330, 200, 0, 129]
    pages = _pages(lengths, kv, hd, ps, fmt, dtype)
    _fill(pages, lengths, dtype)
    bounds = _new_bounds(pages, dtype)
    n, f = torch.tensor(lengths, device=DEV), torch.tensor(first, device=DEV)
    assert paged.summarise(pages, bounds, n, first=f) is None
    want = _new_bounds(pages, dtype)
    for b, (m, lo) in enumerate(zip(lengths, first)):
        for j in range(lo // ps, -(-m // ps) if m > lo else 0):
            at = torch.arange(j * ps, min(m, j * ps + ps), device=DEV)
            k, _ = paged.read(pages, torch.full_like(at, b, dtype=torch.int32), at,
                              torch.float32 if fmt != "same" else None)
            want[pages.table[b, j]] = torch.stack((k.amin(0), k.amax(0)), 1).to(want.dtype)
    assert torch.equal(bounds, want)
    # the same sequences in another order, all of their tokens
    order = torch.tensor([4, 3, 6, 1], dtype=torch.int32, device=DEV)
    paged.summarise(pages, bounds, n[order.long()], seq=order)
    for b in order.tolist():
        at = torch.arange(lengths[b], device=DEV)
        k, _ = paged.read(pages, torch.full_like(at, b, dtype=torch.int32), at, torch.float32 if fmt != "same" else None)
        got = bounds[pages.table[b, : -(-lengths[b] // ps)].long()]
        low, high = got[:, :, 0].amin(0), got[:, :, 1].amax(0)
        assert torch.equal(low, k.amin(0).to(low.dtype)) and torch.equal(high, k.amax(0).to(low.dtype))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_bounds_that_are_not_finite(dtype):
    """Infinities are held as the largest finite value, NaN stays in its own place."""
    from epure import paged
    pages = _pages([16], 1, 32, 16, "same", dtype)
    seq, pos = _tokens([16])
    k = torch.randn(16, 1, 32, generator=_gen(1), device=DEV).to(dtype)
    k[3, 0, 1] = math.inf
    k[5, 0, 2] = -math.inf
    k[6, 0, 3] = math.nan
    k[:, 0, 4] = math.inf
    paged.write(pages, k, k, seq, pos)
    bounds = _new_bounds(pages, dtype)
    paged.summarise(pages, bounds, torch.tensor([16], device=DEV))
    low, high = bounds[pages.table[0, 0]][0]
    top = torch.finfo(dtype).max
    want_low, want_high = k[:, 0].amin(0).clamp(-top, top), k[:, 0].amax(0).clamp(-top, top)
    assert torch.equal(torch.nan_to_num(low, nan=123.0), torch.nan_to_num(want_low, nan=123.0))
    assert torch.equal(torch.nan_to_num(high, nan=123.0), torch.nan_to_num(want_high, nan=123.0))
    assert bool(low[3].isnan()) and int(bounds[pages.table[0, 0]].isnan().sum()) == 2


def test_bounds_of_shared_pages_and_of_a_layer():
    """Rows with a page in common that agree about it, and bounds that are a slice of a larger tensor."""
    from epure import paged
    cache = paged.PagedKVCache(2, 8, 16, 2, 64, seqs=3, max_tokens=64, device=DEV, bounds=True)
    cache.reserve(0, 40)
    assert cache.share(1, 0, 40) == 32 and cache.share(2, 0, 40) == 32
    cache.reserve(1, 40)
    cache.reserve(2, 64)
    lengths = torch.tensor([40, 37, 64], device=DEV)
    x = torch.randn(136, 2, 64, generator=_gen(2), device=DEV).to(torch.bfloat16)
    for layer in range(2):
        pages = cache.layer(layer)
        at, pos = _tokens([40, 40, 64])
        paged.write(pages, x[:40], x[:40], at[:40], pos[:40])
        own = torch.cat((torch.arange(72, 80), torch.arange(112, 144))).to(DEV)
        paged.write(pages, x[:40], x[:40], at[own], pos[own])
        bounds = cache.bounds[layer]
        paged.summarise(pages, bounds, lengths)
        for b, n in enumerate(lengths.tolist()):
            for j in range(-(-n // 16)):
                t = torch.arange(j * 16, min(n, j * 16 + 16), device=DEV)
                k, _ = paged.read(pages, torch.full_like(t, b, dtype=torch.int32), t)
                assert torch.equal(bounds[pages.table[b, j]], torch.stack((k.amin(0), k.amax(0)), 1))


# -- selection ---------------------------------------------------------------------------------------------------

def _score(q, low, high):
    """The documented float32 score of one row's blocks: q [heads, hd], low / high [blocks, hd]."""
    t = torch.maximum(q[:, None] * low, q[:, None] * high)
    t = torch.nn.functional.pad(t, (0, (1 << (t.shape[-1] - 1).bit_length()) - t.shape[-1]))
    while t.shape[-1] > 1:
        t = t[..., 0::2] + t[..., 1::2]
    return t[..., 0].amax(0)                           # (amax passes NaN on)


def _expected(q, bounds, table, n, count, sinks, recent, kv):
    """Lists by sorting: NaN first, then the score, then the lowest block."""
    got = torch.full((q.shape[0], kv, count), -1, dtype=torch.int32)
    g = q.shape[1] // kv
    for b, blocks in enumerate(n):
        edge = bounds[table[b, :blocks].long()].float()
        for h in range(kv):
            score = _score(q[b, h * g:h * g + g].float(), edge[:, h, 0], edge[:, h, 1]).tolist()
            forced = [j for j in range(blocks) if j < sinks or j >= blocks - recent]
            rest = sorted((j for j in range(blocks) if not (j < sinks or j >= blocks - recent)),
                          key=lambda j: (not math.isnan(score[j]), -score[j], j))
            pick = sorted(forced + rest[:max(0, count - len(forced))])
            got[b, h, :len(pick)] = torch.tensor(pick, dtype=torch.int32)
    return got.to(DEV)


def _selection_case(heads, kv, hd, n, fmt="same", dtype=torch.bfloat16, seed=3, ps=16):
    lengths = [max(0, m * ps - i % ps) for i, m in enumerate(n)]
    pages = _pages(lengths, kv, hd, ps, fmt, dtype)
    g = _gen(seed)
    mid = torch.randn(pages.k.shape[0], kv, hd, generator=g, device=DEV)
    half = torch.rand(mid.shape, generator=g, device=DEV) * 2
    bounds = torch.stack((mid - half, mid + half), 2).to(dtype if fmt == "same" else torch.bfloat16)
    q = torch.randn(len(n), heads, hd, generator=g, device=DEV).to(dtype)
    return pages, bounds, q, torch.tensor(lengths, device=DEV)


@pytest.mark.parametrize("heads,kv,hd", [(32, 8, 128), (8, 8, 64), (4, 2, 128), (12, 4, 80), (28, 4, 128), (16, 1, 64), (6, 2, 256),
                                         (40, 2, 48), (3, 1, 16), (24, 2, 256)])
@pytest.mark.parametrize("fmt,dtype", [("same", torch.bfloat16), ("same", torch.float16), ("int8", torch.bfloat16),
                                       ("fp8", torch.float16)])
def test_select(heads, kv, hd, fmt, dtype):
    from epure import paged
    n = [1, 0, 5, 6, 7, 64, 65, 300]
    pages, bounds, q, lengths = _selection_case(heads, kv, hd, n, fmt, dtype)
    for count, sinks, recent in ((6, 1, 1), (5, 0, 0), (64, 2, 3), (4, 3, 1), (1, 0, 0), (400, 1, 1)):
        got = paged.select(pages, bounds, q, lengths, count, sinks=sinks, recent=recent)
        assert torch.equal(got, _expected(q, bounds, pages.table, n, count, sinks, recent, kv)), (count, sinks, recent)


@pytest.mark.parametrize("blocks", [1023, 4096, 4097, 9000])
def test_select_many_blocks(blocks):
    """Scores of more blocks than a CTA's registers hold (4,096), cut over many CTAs."""
    from epure import paged
    pages, bounds, q, lengths = _selection_case(8, 2, 64, [blocks], ps=1)
    for count in (1, 77, 1000):
        got = paged.select(pages, bounds, q, lengths, count, sinks=1, recent=0)
        assert torch.equal(got, _expected(q, bounds, pages.table, [blocks], count, 1, 0, 2))
        assert torch.equal(paged.select(pages, bounds, q, lengths, count, sinks=1, recent=0), got)


def test_select_ties_and_not_finite_scores():
    """Equal scores go to the lowest block; a block with NaN comes first, infinities are in order, -0 is 0."""
    from epure import paged
    pages, bounds, q, lengths = _selection_case(4, 2, 64, [200, 130])
    bounds.copy_(bounds.sign())                        # few different scores
    q = torch.where(q > 0, 1.0, -1.0).to(torch.bfloat16) * (torch.arange(64, device=DEV) < 4)
    for count in (3, 20, 129):
        got = paged.select(pages, bounds, q, lengths, count, sinks=0, recent=1)
        assert torch.equal(got, _expected(q, bounds, pages.table, [200, 130], count, 0, 1, 2))
    bounds[pages.table[0, 150].long(), 0, 1, 3] = math.nan
    bounds[pages.table[0, 7].long(), 1] = 3e38         # sums of +inf
    bounds[pages.table[0, 60].long(), 1] = 3e38
    bounds[pages.table[1, 4].long()] = 0.0
    bounds[pages.table[1, 9].long()] = -0.0
    q = q + 1.5
    for count in (2, 3, 40):
        got = paged.select(pages, bounds, q, lengths, count, sinks=0, recent=1)
        want = _expected(q, bounds, pages.table, [200, 130], count, 0, 1, 2)
        assert torch.equal(got, want)
    assert 150 in got[0, 0].tolist() and 7 in got[0, 1].tolist()
    q.fill_(0)                                         # all scores 0: the lowest blocks
    got = paged.select(pages, torch.zeros_like(bounds), q, lengths, 10, sinks=0, recent=1)
    assert got[0, 0].tolist() == list(range(9)) + [199] and got[1, 1].tolist() == list(range(9)) + [129]


@pytest.mark.parametrize("blocks,nans", [(60, 20), (300, 12), (300, 299), (5000, 20), (9000, 1500)])
@pytest.mark.parametrize("fmt,dtype", [("same", torch.bfloat16), ("same", torch.float16), ("int8", torch.float16)])
def test_select_as_many_nan_as_are_wanted(blocks, nans, fmt, dtype):
    """Blocks with NaN come first, the lowest of them, be there more than are wanted, as many or fewer."""
    from epure import paged
    n = [blocks, 40, blocks]
    pages, bounds, q, lengths = _selection_case(4, 2, 64, n, fmt, dtype, ps=1)
    pick = torch.randperm(blocks - 2, generator=torch.Generator().manual_seed(blocks))[:nans] + 1
    for h, d in ((0, 5), (1, 63)):
        bounds[pages.table[0, pick.to(DEV)].long(), h, h, d] = math.nan
    q[2, 1, 7] = math.nan                              # all scores of a key head
    for count in sorted({2, nans // 2 + 3, nans + 2, min(blocks - 1, nans + 9)}):
        got = paged.select(pages, bounds, q, lengths, count)
        assert torch.equal(got, _expected(q, bounds, pages.table, n, count, 1, 1, 2)), count


@pytest.mark.parametrize("fmt,cache,dtype", [("same", torch.bfloat16, torch.bfloat16), ("same", torch.float16, torch.float16),
                                             ("int8", torch.bfloat16, torch.float16), ("same", torch.float16, torch.bfloat16)])
@pytest.mark.parametrize("heads,kv,hd,blocks", [(8, 1, 128, 300), (24, 2, 64, 900), (6, 2, 256, 130), (4, 4, 80, 3000)])
def test_select_scores_apart_by_their_rounding(fmt, cache, dtype, heads, kv, hd, blocks):
    """Blocks that differ in the last bits of their sums, of up to 1024 and of more: the defined order of summing decides."""
    from epure import paged
    pages, bounds, q, lengths = _selection_case(heads, kv, hd, [blocks, 40], fmt, cache, ps=1)
    q = q.to(dtype)
    bounds[:, :, :, 1:] = bounds[:1, :, :, 1:]                                 # all alike...
    bounds[:, :, :, 0] = 100.0
    small = torch.rand(bounds.shape[0], kv, 2, hd // 4, generator=_gen(8), device=DEV) * 2e-3
    bounds[..., hd // 2:hd // 2 + hd // 4] = (small.sort(2).values + 1e-3).to(bounds.dtype)    # ... but for these
    for count in (2, 33, 120):
        got = paged.select(pages, bounds, q, lengths, count)
        assert torch.equal(got, _expected(q, bounds, pages.table, [blocks, 40], count, 1, 1, kv)), count


@pytest.mark.parametrize("fmt,cache,dtype", [("same", torch.bfloat16, torch.bfloat16), ("int8", torch.bfloat16, torch.float16),
                                             ("same", torch.float16, torch.bfloat16)])
def test_select_queries_of_any_size(fmt, cache, dtype):
    """Queries near both ends of their type's range, and of both in one row."""
    from epure import paged
    pages, bounds, q, lengths = _selection_case(8, 2, 64, [90] * 6, fmt, cache)
    q = q.to(dtype)
    large, small = (3e4, 1e-7) if dtype == torch.float16 else (1e37, 1e-39)
    q[0] *= large / 8
    q[1] *= small
    q[2, :, ::3] *= large / 8
    q[3, ::2] *= small
    q[4, 1] = 0
    q[5, :, 5:] *= 0
    got = paged.select(pages, bounds, q, lengths, 12)
    assert torch.equal(got, _expected(q, bounds, pages.table, [90] * 6, 12, 1, 1, 2))


def test_select_other_layouts():
    """Rows of a projection, rows that are not aligned, a subset of the sequences, several rows of one."""
    from epure import paged
    pages, bounds, q, lengths = _selection_case(8, 2, 128, [40, 90, 17])
    want = paged.select(pages, bounds, q, lengths, 8)
    wide = torch.zeros(3, 12, 128, dtype=q.dtype, device=DEV)
    wide[:, 2:10] = q
    assert torch.equal(paged.select(pages, bounds, wide[:, 2:10], lengths, 8), want)
    odd = torch.empty(q.numel() + 1, dtype=q.dtype, device=DEV)[1:].view(q.shape).copy_(q)
    assert torch.equal(paged.select(pages, bounds, odd, lengths, 8), want)
    swap = torch.empty(8, 3, 128, dtype=q.dtype, device=DEV).transpose(0, 1).copy_(q)
    assert torch.equal(paged.select(pages, bounds, swap, lengths, 8), want)
    pick = torch.tensor([2, 1, 1], dtype=torch.int32, device=DEV)
    got = paged.select(pages, bounds, q[[2, 1, 0]], torch.tensor([int(lengths[2]), int(lengths[1]), 33 * 16], device=DEV), 8,
                       seq=pick)
    assert torch.equal(got[0], want[2]) and torch.equal(got[1], want[1])
    assert torch.equal(got[2:], _expected(q[:1], bounds, pages.table[1:2], [33], 8, 1, 1, 2))
    spread = torch.zeros(bounds.shape[0], 2, *bounds.shape[1:], dtype=bounds.dtype, device=DEV)
    spread[:, 1] = bounds
    assert torch.equal(paged.select(pages, spread[:, 1], q, lengths, 8), want)


# -- attention over listed blocks --------------------------------------------------------------------------------

def _check_listed(pages, q, lengths, blocks, k, v, seq=None, scale=None):
    """Against 64 bits, head by head; the bounds are those of attention over all tokens."""
    from epure import paged
    B, H, hd = q.shape
    kv, ps = pages.k.shape[1], pages.k.shape[2]
    sc = 1 / math.sqrt(hd) if scale is None else scale
    out, lse = paged.attend(pages, q, torch.tensor(lengths, device=DEV), seq=seq, scale=scale, blocks=blocks, return_lse=True)
    unit = UNIT[torch.float16] if pages.k_scale is not None else UNIT[q.dtype]
    starts = [sum(lengths[:b]) for b in range(B)]
    for b, n in enumerate(lengths):
        for g in range(kv):
            listed = [j for j in blocks[b, g, :-(-n // ps)].tolist() if j >= 0]
            at = [t for j in listed for t in range(j * ps, min(n, j * ps + ps))]
            hs = slice(g * (H // kv), (g + 1) * (H // kv))
            if not at:
                assert not out[b, hs].any() and bool(torch.isneginf(lse[b, hs]).all())
                continue
            kk, vv = (x[torch.tensor(at, device=DEV) + starts[b], g] for x in (k, v))
            z = q[b, hs].double() @ kk.T * sc
            p = torch.softmax(z, -1)
            want, mag = p @ vv, p @ vv.abs()
            err = 2.0 ** -23 * (hd * (q[b, hs].double().abs() @ kk.abs().T).amax(-1) * sc + 4 * z.abs().amax(-1))
            small = 2.0 ** -25 * len(at) * float(vv.abs().max()) if unit == 2.0 ** -11 else 0.0
            bound = UNIT[q.dtype] * want.abs() + (unit + 2 * err[:, None] + 2.0 ** -18) * 1.01 * mag + small + 2.0 ** -25
            assert bool(((out[b, hs].double() - want).abs() <= bound).all()), (b, g)
            exact = torch.logsumexp(z, -1)
            assert bool(((lse[b, hs].double() - exact).abs() <= err + 2.0 ** -20 * (1 + exact.abs())).all())
    return out, lse


@pytest.mark.parametrize("fmt", ["same", "int8", "fp8"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("heads,kv,hd,ps", [(32, 8, 128, 16), (8, 2, 64, 64), (12, 4, 80, 24), (28, 4, 128, 7), (16, 1, 64, 1),
                                            (40, 2, 64, 48), (6, 2, 256, 16), (3, 3, 16, 5)])
def test_attend_listed(fmt, dtype, heads, kv, hd, ps):
    """Random lists in random orders, holes among them, empty ones, and more entries than a row has blocks."""
    lengths = [0, 1, 16, 65, 333, 1000, 64, 200]
    pages = _pages(lengths, kv, hd, ps, fmt, dtype)
    k, v = _fill(pages, lengths, dtype)
    q = (torch.randn(len(lengths), heads, hd, generator=_gen(7), device=DEV) * 2).to(dtype)
    g = torch.Generator().manual_seed(8)
    count = 12
    blocks = torch.full((len(lengths), kv, count), -1, dtype=torch.int32)
    for b, n in enumerate(lengths):
        for h in range(kv):
            pick = torch.randperm(max(1, -(-n // ps)), generator=g)[:count].int()
            pick[torch.rand(pick.shape, generator=g) < 0.2] = -1
            blocks[b, h, :len(pick)] = pick
    blocks[5, 0] = -1
    blocks[6, :, -(-64 // ps):] = 10 ** 6              # entries behind what a row has are not looked at
    blocks = blocks.to(DEV)
    one = _check_listed(pages, q, lengths, blocks, k, v)
    two = _check_listed(pages, q, lengths, blocks, k, v)
    assert torch.equal(one[0], two[0]) and torch.equal(one[1], two[1])


def test_attend_all_blocks_listed():
    """Lists of all blocks give what attention without a list gives, within its bounds."""
    lengths = [5000, 64, 1, 777]
    pages = _pages(lengths, 4, 128, 16, "int8", torch.bfloat16)
    k, v = _fill(pages, lengths, torch.bfloat16)
    q = torch.randn(4, 16, 128, generator=_gen(9), device=DEV).to(torch.bfloat16)
    blocks = torch.arange(pages.table.shape[1], dtype=torch.int32, device=DEV).expand(4, 4, -1).contiguous()
    _check_listed(pages, q, lengths, blocks, k, v)


def test_attend_listed_more_units_than_ctas():
    """Runs that go over unit boundaries, empty rows between."""
    lengths = [0, 40, 300, 7] * 40
    pages = _pages(lengths, 8, 64, 16, "same", torch.bfloat16)
    k, v = _fill(pages, lengths, torch.bfloat16)
    q = torch.randn(len(lengths), 16, 64, generator=_gen(10), device=DEV).to(torch.bfloat16)
    blocks = torch.tensor([[3, 0, 11, -1, 18], [18, 5, 4, 1, 0]], dtype=torch.int32).repeat(len(lengths), 4, 1)
    blocks = torch.where(blocks * 16 < torch.tensor(lengths)[:, None, None], blocks, -1).to(DEV)
    _check_listed(pages, q, lengths, blocks, k, v)


def test_no_blocks():
    from epure import paged
    pages = _pages([30], 2, 64, 16, "same", torch.bfloat16)
    _fill(pages, [30], torch.bfloat16)
    q = torch.randn(1, 4, 64, device=DEV).to(torch.bfloat16)
    out, lse = paged.attend(pages, q, torch.tensor([30], device=DEV), return_lse=True,
                            blocks=torch.empty(1, 2, 0, dtype=torch.int32, device=DEV))
    assert not out.any() and bool(torch.isneginf(lse).all())
    empty = paged.select(pages, _new_bounds(pages, torch.bfloat16), q[:0], torch.empty(0, dtype=torch.long, device=DEV), 4)
    assert empty.shape == (0, 2, 4)


# -- together ----------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("fmt", ["same", "int8"])
def test_a_step_captured(fmt):
    """Write, bounds, selection and attention in one graph, replayed as the sequences grow and a page begins, on another
    stream than the one it was captured on; equal to the same calls outside it."""
    from epure import paged
    KV, H, hd, ps = 2, 8, 64, 16
    def fresh():
        cache = paged.PagedKVCache(1, 64, ps, KV, hd, seqs=2, max_tokens=400, format=fmt, device=DEV, bounds=True)
        cache.reserve(0, 400)
        cache.reserve(1, 130)
        at, pos = _tokens([250, 95])
        x = torch.randn(345, KV, hd, generator=_gen(12), device=DEV).to(torch.bfloat16)
        paged.write(cache.layer(0), x, x.flip(0), at, pos)
        paged.summarise(cache.layer(0), cache.bounds[0], torch.tensor([250, 95], device=DEV))
        return cache

    def step(cache, qkv, pos, seq):
        pages = cache.layer(0)
        paged.write(pages, qkv[:, H:H + KV], qkv[:, H + KV:], seq, pos)
        n = pos + 1
        paged.summarise(pages, cache.bounds[0], n, seq=seq, first=pos)
        chosen = paged.select(pages, cache.bounds[0], qkv[:, :H], n, 6, seq=seq)
        return paged.attend(pages, qkv[:, :H], n, seq=seq, blocks=chosen, return_lse=True) + (chosen,)

    rows = torch.randn(10, 2, H + 2 * KV, hd, generator=_gen(13), device=DEV).to(torch.bfloat16)
    seq = torch.arange(2, dtype=torch.int32, device=DEV)
    eager, captured = fresh(), fresh()
    qkv, pos = rows[0].clone(), torch.tensor([250, 95], device=DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(captured, qkv, pos, seq)                  # (written again by the first replay)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(captured, qkv, pos, seq)
    for t in range(10):
        qkv.copy_(rows[t])
        pos.copy_(torch.tensor([250 + t, 95 + t], device=DEV))
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            graph.replay()
        want = step(eager, rows[t], torch.tensor([250 + t, 95 + t], device=DEV), seq)
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b)
        assert torch.equal(captured.bounds, eager.bounds)


def test_refusals():
    from epure import paged
    pages = _pages([30, 5], 2, 64, 16, "same", torch.bfloat16)
    _fill(pages, [30, 5], torch.bfloat16)
    bounds = _new_bounds(pages, torch.bfloat16)
    q = torch.randn(2, 4, 64, device=DEV).to(torch.bfloat16)
    n = torch.tensor([30, 5], device=DEV)
    blocks = torch.zeros(2, 2, 3, dtype=torch.int32, device=DEV)
    for bad in (bounds.half(), bounds.cpu(), bounds[1:], bounds[:, :1], bounds.transpose(2, 3), bounds[..., :32]):
        with pytest.raises(RuntimeError, match="bounds must be"):
            paged.summarise(pages, bad, n)
        with pytest.raises(RuntimeError, match="bounds must be"):
            paged.select(pages, bad, q, n, 4)
    for kw in (dict(count=0), dict(count=3, sinks=2, recent=2), dict(count=3, sinks=-1), dict(count=3, recent=-1)):
        with pytest.raises(RuntimeError, match="count"):
            paged.select(pages, bounds, q, n, **kw)
    with pytest.raises(TypeError, match="queries"):
        paged.select(pages, bounds, q.float(), n, 4)
    with pytest.raises(RuntimeError, match="query heads"):
        paged.select(pages, bounds, q[:, :3], n, 4)
    with pytest.raises(RuntimeError, match="lengths"):
        paged.select(pages, bounds, q, n[:1], 4)
    with pytest.raises(RuntimeError, match="first"):
        paged.summarise(pages, bounds, n, first=n.int())
    with pytest.raises(RuntimeError, match="seq"):
        paged.summarise(pages, bounds, n, seq=n)
    with pytest.raises(RuntimeError, match="table of"):
        paged.summarise(pages, bounds, torch.cat((n, n)))
    for bad in (blocks.long(), blocks[:1], blocks[:, :1], blocks.cpu(), blocks.transpose(1, 2), blocks[..., ::2]):
        with pytest.raises(RuntimeError, match="blocks must be"):
            paged.attend(pages, q, n, blocks=bad)
    with pytest.raises(RuntimeError, match="window"):
        paged.attend(pages, q, n, blocks=blocks, window=5)
    with pytest.raises(RuntimeError, match="gradient"):
        paged.summarise(pages, bounds.clone().requires_grad_(), n)
    plain = _pages([30], 2, 64, 16, "same", torch.float32)
    with pytest.raises(TypeError, match="float32"):
        paged.summarise(plain, bounds, n[:1])
    version = bounds._version
    paged.summarise(pages, bounds, n)
    assert bounds._version == version + 1


_CHILD = r"""
import sys, torch
sys.path.insert(0, sys.argv[1])
from epure import _native, paged
dev, kind = "cuda:0", sys.argv[2]
k = torch.randn(8, 2, 16, 64, device=dev).to(torch.bfloat16)
pages = paged.KVPages(k, k.clone(), torch.tensor([[0, 1, 4, 5], [2, 9, 3, 6]], dtype=torch.int32, device=dev))
q = torch.randn(2, 4, 64, device=dev).to(torch.bfloat16)
t = lambda *v: torch.tensor(v, device=dev)
bounds = torch.full((8, 2, 2, 64), 5.0, device=dev).to(torch.bfloat16)
blocks = torch.tensor([[0, 2], [1, 3]], dtype=torch.int32, device=dev).repeat(2, 1, 1)
paged.summarise(pages, bounds, t(64), seq=t(0).int())
assert _native.device_error() == 0
keep = bounds.clone()
if kind == "bounds-length":
    paged.summarise(pages, bounds, t(65, -1))
    assert torch.equal(bounds, keep)
elif kind == "bounds-first":
    paged.summarise(pages, bounds, t(64), first=t(-1))
    assert torch.equal(bounds, keep)
elif kind == "bounds-seq":
    paged.summarise(pages, bounds, t(16), seq=t(2).int())
    assert torch.equal(bounds, keep)
elif kind == "bounds-page":
    paged.summarise(pages, bounds, t(64), seq=t(1).int())
    assert torch.equal(bounds[[0, 1, 4, 5, 7]], keep[[0, 1, 4, 5, 7]]) and not (bounds[[2, 3, 6]] == 5).any()
elif kind == "select-length":
    got = paged.select(pages, bounds, q, t(65, 16), 2)
    assert (got[0] == -1).all()
elif kind == "select-page":                            # a block outside the pool comes last
    got = paged.select(pages, bounds, q, t(64, 64), 3, sinks=0, recent=0)
    assert (got[1] == t(0, 2, 3).int()).all()
elif kind == "attend-block":
    blocks[0, 0, 1] = 4
    out, lse = paged.attend(pages, q, t(64, 16), blocks=blocks, return_lse=True)
    blocks[0, 0, 1] = -1
    want = paged.attend(pages, q, t(64, 16), blocks=blocks, return_lse=True)
    assert torch.equal(out, want[0]) and torch.equal(lse, want[1])
elif kind == "attend-page":
    out = paged.attend(pages, q, t(64, 64), blocks=blocks)
    blocks[1, 1, 0] = -1
    want = paged.attend(pages, q, t(64, 64), blocks=blocks)
    assert torch.equal(out, want)
torch.cuda.synchronize()
print("FLAG", _native.device_error())
"""


@pytest.mark.parametrize("kind,flag", [("bounds-length", 16), ("bounds-first", 16), ("bounds-seq", 16), ("bounds-page", 32),
                                       ("select-length", 16), ("select-page", 32), ("attend-block", 16), ("attend-page", 32)])
def test_bad_lengths_blocks_and_pages_are_reported(kind, flag):
    """Skipped and reported by epq_device_error (in a child process: the flag stays set)."""
    r = subprocess.run([sys.executable, "-c", _CHILD, PKG, kind], capture_output=True, text=True, timeout=300,
                       env=dict(os.environ))
    assert r.returncode == 0, r.stderr[-2000:]
    assert f"FLAG {flag}" in r.stdout
