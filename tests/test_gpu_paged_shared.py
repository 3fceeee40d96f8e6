"""Attention of rows that share a prefix (paged.attend_shared) against 64 bits, and what the plan makes of the groups."""
import math
import os
import subprocess
import sys

import pytest
import torch
from conftest import PKG
from test_gpu_paged import DEV, UNIT, _gen, _gpu, _reference  # noqa: F401 (_gpu: a fixture)

pytestmark = pytest.mark.gpu


def _case(groups, kv, hd, ps, fmt, dtype, seed=0, same=False, scale_range=0.0, spare=3):
    """A filled cache, starts, prefix, seq, lengths, and per row the tokens that it sees as 64-bit (k, v).

    ``groups``: (prefix, own tokens of each row, -1 for an empty row).  Rows are sequences of their own behind shared pages,
    or with ``same`` several rows of the group's one sequence.  Slots that are no token hold NaN."""
    from epure import paged
    g = _gen(seed)
    need, share, rows, lengths, starts, prefix = [], [], [], [], [0], []
    for p, own in groups:
        first = len(need)
        if same:
            need.append(p + max(own + [0]))
            share.append(None)
            rows += [first] * len(own)
        else:
            for i, n in enumerate(own):
                need.append(p + max(n, 0))
                share.append((first, p // ps) if i else None)
                rows.append(first + i)
        lengths += [p + n if n >= 0 else 0 for n in own]
        starts.append(starts[-1] + len(own))
        prefix.append(p)
    whole = [s[1] if s else 0 for s in share]
    total = sum(-(-n // ps) - w for n, w in zip(need, whole)) + spare
    order = torch.randperm(total, generator=g, device=DEV).int().cpu()
    table = torch.full((len(need), max(1, max(-(-n // ps) for n in need))), -1, dtype=torch.int32)
    at = 0
    for i, n in enumerate(need):
        if share[i]:
            table[i, :whole[i]] = table[share[i][0], :whole[i]]
        more = -(-n // ps) - whole[i]
        table[i, whole[i]:whole[i] + more] = order[at:at + more]
        at += more
    kinds = {"same": dtype, "int8": torch.int8, "fp8": torch.float8_e4m3fn}
    shape = (total, kv, ps, hd)
    nan = float("nan")
    if fmt == "same":
        pages = paged.KVPages(torch.full(shape, nan, dtype=dtype, device=DEV), torch.full(shape, nan, dtype=dtype, device=DEV),
                              table.to(DEV))
    else:
        codes = [torch.full(shape, 0x7f, dtype=torch.int8, device=DEV).view(kinds[fmt]) for _ in range(2)]
        pages = paged.KVPages(*codes, table.to(DEV), torch.full(shape[:3], nan, device=DEV), torch.full(shape[:3], nan, device=DEV))
    # tokens: a prefix's are the same in all of its rows, wherever they lie
    ks, vs = [], []
    shared = {}
    for i, n in enumerate(need):
        k, v = (torch.randn(n, kv, hd, generator=g, device=DEV) for _ in range(2))
        if scale_range:
            v *= torch.exp2(scale_range * (2 * torch.rand(n, kv, 1, generator=g, device=DEV) - 1))
        first = share[i][0] if share[i] else i
        if share[i]:
            pre = prefix[[j for j, s in enumerate(starts[1:]) if s > i][0]]
            k[:pre], v[:pre] = shared[first][0][:pre], shared[first][1][:pre]
        else:
            shared[i] = (k, v)
        ks.append(k.to(dtype))
        vs.append(v.to(dtype))
    at = torch.cat([torch.full((n,), i, dtype=torch.int32) for i, n in enumerate(need)]).to(DEV)
    pos = torch.cat([torch.arange(n) for n in need]).to(DEV)
    new = torch.cat([torch.arange(n) >= w * ps for n, w in zip(need, whole)]).to(DEV)   # (shared pages are written once)
    if len(pos):
        kk, vv = torch.cat(ks), torch.cat(vs)
        paged.write(pages, kk[new], vv[new], at[new], pos[new])
        if fmt != "same":
            kk, vv = paged.read(pages, at, pos, torch.float32)
        ks, vs = list(kk.double().split(need)), list(vv.double().split(need))
    seq = torch.tensor(rows, dtype=torch.int32, device=DEV)
    seen = [(ks[r][:n], vs[r][:n]) for r, n in zip(rows, lengths)]
    return pages, torch.tensor(starts, dtype=torch.int32, device=DEV), torch.tensor(prefix, device=DEV), seq, lengths, seen


def _check(case, q, scale=None, **kw):
    """The bounds of attention without sharing (two parts of a weight keep 16 bits in bf16, so one rounding covers them);
    8-bit caches' weights are bf16 pairs here."""
    from epure import paged
    pages, starts, prefix, seq, lengths, seen = case
    sc = 1 / math.sqrt(q.shape[-1]) if scale is None else scale
    n = torch.tensor(lengths, device=DEV)
    out, lse = paged.attend_shared(pages, q, n, starts, prefix, seq=seq, scale=scale, return_lse=True, **kw, always=True)
    again = paged.attend_shared(pages, q, n, starts, prefix, seq=seq, scale=scale, return_lse=True, always=True)
    assert torch.equal(out, again[0]) and torch.equal(lse, again[1])           # the order of the pieces is fixed
    k = torch.cat([s[0] for s in seen]).double()
    v = torch.cat([s[1] for s in seen]).double()
    want, want_lse, mag, err = _reference(q, k, v, lengths, 0, abs(sc)) if sc >= 0 else _reference(-q, k, v, lengths, 0, -sc)
    unit = UNIT[torch.float16] if pages.k_scale is not None else UNIT[q.dtype]
    small = 2.0 ** -25 * max(lengths) * float(v.abs().max()) if unit == 2.0 ** -11 and v.numel() else 0.0
    bound = UNIT[q.dtype] * want.abs() + (unit + 2 * err[..., None] + 2.0 ** -18) * 1.01 * mag + small + 2.0 ** -25
    off = (out.double() - want).abs()
    assert bool((off <= bound).all()), (float((off / bound).max()), int((off > bound).sum()))
    empty = torch.isinf(want_lse)
    assert torch.equal(torch.isneginf(lse), empty) and not out[empty].any()
    off = (lse.double() - want_lse)[~empty].abs()
    assert bool((off <= err[~empty] + 2.0 ** -20 * (1 + want_lse[~empty].abs())).all()), float(off.max())
    return out, lse


def _q(case, heads, hd, dtype, seed=5, gain=2.0):
    return (torch.randn(len(case[4]), heads, hd, generator=_gen(seed), device=DEV) * gain).to(dtype)


LONG = [(9000, [0, 5, 100, -1, 300, 17, 64, 1] * 3), (4000, [3, 0]), (1, [5, 9]), (0, [1, -1, 40]), (2049, [-1, -1, -1]),
        (2500, [8] * 11), (6000, [])]


@pytest.mark.parametrize("fmt", ["same", "int8", "fp8"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("heads,kv,hd,ps", [(32, 8, 128, 64), (8, 8, 128, 16), (64, 4, 128, 48), (12, 4, 80, 24), (8, 2, 64, 7),
                                            (16, 1, 64, 128), (3, 3, 16, 1), (28, 4, 112, 32), (6, 2, 256, 16), (40, 1, 192, 64)])
def test_prompts(fmt, dtype, heads, kv, hd, ps):
    """Ragged groups of sequences behind a common prefix: empty rows, empty groups, rows without own tokens, groups of one
    tile and of several, prefixes that end inside a page."""
    case = _case(LONG, kv, hd, ps, fmt, dtype)
    _check(case, _q(case, heads, hd, dtype))


@pytest.mark.parametrize("fmt", ["same", "int8", "fp8"])
@pytest.mark.parametrize("heads,kv,hd,ps", [(32, 8, 128, 64), (16, 8, 128, 16), (12, 4, 80, 24), (8, 2, 256, 16)])
def test_drafts_and_chunks(fmt, heads, kv, hd, ps):
    """Rows of one sequence with lengths of their own: drafted tokens, and a prompt's chunk of more rows than a tile."""
    groups = [(5000, [1, 2, 3, 4, 5]), (8191, [1, 2, 3]), (300, [1]), (3000, list(range(1, 300))), (0, list(range(1, 40)))]
    case = _case(groups, kv, hd, ps, fmt, torch.bfloat16, same=True)
    _check(case, _q(case, heads, hd, torch.bfloat16))


@pytest.mark.parametrize("fmt", ["same", "fp8"])
def test_prefix_longer_than_rows(fmt):
    """A prefix that reaches past some rows' lengths: they see their own tokens alone, whatever lies behind."""
    groups = [(9000, [1, 2, 3, 4] * 8)]
    pages, starts, prefix, seq, lengths, seen = _case(groups, 4, 128, 64, fmt, torch.bfloat16, same=True)
    lengths = [n - 37 * i for i, n in enumerate(lengths)]
    seen = [(k[:n], v[:n]) for (k, v), n in zip(seen, lengths)]
    for p in (9004, 8500, 40):
        case = (pages, starts, torch.tensor([p], device=DEV), seq, lengths, seen)
        _check(case, _q(case, 16, 128, torch.bfloat16))


def test_one_prefix_many_rows():
    """More units than CTAs, whole and cut ones, and a batch whose rows all stop at the prefix."""
    case = _case([(3000, [i % 5 for i in range(700)])], 8, 64, 16, "same", torch.bfloat16)
    _check(case, _q(case, 16, 64, torch.bfloat16))
    case = _case([(20011, [0] * 40)], 2, 128, 64, "int8", torch.bfloat16)
    _check(case, _q(case, 16, 128, torch.bfloat16))


def test_agrees_with_attention_without_sharing():
    from epure import paged
    case = _case(LONG, 8, 128, 64, "int8", torch.bfloat16)
    pages, starts, prefix, seq, lengths, _ = case
    q = _q(case, 32, 128, torch.bfloat16)
    n = torch.tensor(lengths, device=DEV)
    a, la = paged.attend(pages, q, n, seq=seq, return_lse=True)
    b, lb = paged.attend_shared(pages, q, n, starts, prefix, seq=seq, return_lse=True, always=True)
    # two results within their own rounding of each other, and float32 sums in another order
    assert float((a.double() - b.double()).abs().max()) <= 2.0 ** -7 * float(a.abs().max())
    some = torch.isfinite(la)
    assert torch.equal(some, torch.isfinite(lb)) and float((la - lb)[some].abs().max()) <= 1e-4
    # no group, groups of one row, starts that leave rows out
    for s, p in (([0], []), (list(range(len(lengths) + 1)), [100] * len(lengths)), ([3, 3, 9], [9000, 9000])):
        got = paged.attend_shared(pages, q, n, torch.tensor(s, dtype=torch.int32, device=DEV),
                                  torch.tensor(p, dtype=torch.long, device=DEV), seq=seq, always=True)
        assert float((a.double() - got.double()).abs().max()) <= 2.0 ** -7 * float(a.abs().max())


@pytest.mark.parametrize("fmt", ["same", "int8", "fp8"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_uneven_scores_and_scales(fmt, dtype):
    """Peaks that keep rising along the prefix, value rows apart by 2^24, scales of 0, large and below 0."""
    case = _case([(9000, [7, 0, 30] * 6)], 2, 64, 16, fmt, dtype, scale_range=12.0 if dtype == torch.bfloat16 else 6.0)
    q = _q(case, 8, 64, dtype, gain=1.0)
    _check(case, q * 12)
    _check(case, q * 1e-3)
    _check(case, q, scale=2.5)
    _check(case, q, scale=0.0)
    _check(case, q, scale=-0.3)


def test_rising_scores_move_the_maximum():
    """Keys that grow along the prefix: every block passes the running maximum by far, in all four warps' rows at different
    places."""
    from epure import paged
    case = _case([(9000, [2] * 40)], 1, 64, 16, "same", torch.bfloat16)
    pages, starts, prefix, seq, lengths, seen = case
    at, pos = torch.zeros(9000, dtype=torch.int32, device=DEV), torch.arange(9000, device=DEV)
    k, v = paged.read(pages, at, pos)
    k = (k.float() * (1 + pos[:, None, None] / 300.0)).to(torch.bfloat16)
    whole = 9000 // 16 * 16
    paged.write(pages, k[:whole], v[:whole], at[:whole], pos[:whole])
    for r, n in enumerate(lengths):                       # the part page of every row
        t = pos[whole:]
        paged.write(pages, k[whole:], v[whole:], torch.full_like(t, r, dtype=torch.int32), t)
    seen = [(torch.cat((k[:9000].double(), s[0][9000:])), s[1]) for s in seen]
    _check((pages, starts, prefix, seq, lengths, seen), _q(case, 8, 64, torch.bfloat16, gain=1.0))


def test_not_finite_values_stay_in_their_row():
    """NaN in a row's own tokens or query, and -inf keys of the prefix that leave weight 0."""
    from epure import paged
    case = _case([(9000, [40, 3, 0, 50] * 5)], 2, 64, 16, "same", torch.bfloat16)
    pages, starts, prefix, seq, lengths, seen = case
    q = _q(case, 8, 64, torch.bfloat16, gain=0.5).abs()
    n = torch.tensor(lengths, device=DEV)
    want = paged.attend_shared(pages, q, n, starts, prefix, seq=seq, always=True)
    t = torch.tensor([9020], device=DEV)
    bad = torch.full((1, 2, 64), float("nan"), dtype=torch.bfloat16, device=DEV)
    paged.write(pages, bad, bad, seq[4:5], t)
    q[9, 3] = float("nan")
    got = paged.attend_shared(pages, q, n, starts, prefix, seq=seq, always=True)
    assert torch.isnan(got[4]).all() and torch.isnan(got[9, 3]).all()
    keep = torch.ones(20, 8, dtype=torch.bool, device=DEV)
    keep[4] = False
    keep[9, 3] = False
    assert torch.equal(got[keep], want[keep])
    # keys of -inf with positive queries
    k = torch.full((1, 2, 64), float("-inf"), dtype=torch.bfloat16, device=DEV)
    v = torch.ones(1, 2, 64, dtype=torch.bfloat16, device=DEV)
    paged.write(pages, k, v, seq[:1], torch.tensor([123], device=DEV))
    out, lse = paged.attend_shared(pages, q.abs() + 0.1, n, starts, prefix, seq=seq, return_lse=True, always=True)
    assert torch.isfinite(out[keep]).all() and torch.isfinite(lse[keep]).all()


def test_a_value_beyond_a_row_stays_unseen():
    """A later row's token that is not finite: rows that end before it do not see it, though a tile holds them all."""
    from epure import paged
    pages, starts, prefix, seq, lengths, seen = _case([(9000, [1, 2, 3, 4, 5, 6])], 2, 128, 64, "same", torch.bfloat16, same=True)
    case = (pages, starts, torch.tensor([9006], device=DEV), seq, lengths, seen)
    q = _q(case, 8, 128, torch.bfloat16)
    bad = torch.full((1, 2, 128), float("inf"), dtype=torch.bfloat16, device=DEV)
    paged.write(pages, bad, bad, seq[:1], torch.tensor([9003], device=DEV))
    n = torch.tensor(lengths, device=DEV)
    got = paged.attend_shared(pages, q, n, starts, case[2], seq=seq, always=True)
    assert torch.isfinite(got[:3]).all() and not torch.isfinite(got[3:]).any()
    case = (pages, starts[:1].new_tensor([0, 3]), case[2], seq[:3], lengths[:3], seen[:3])
    _check(case, q[:3])


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
def test_weights_are_not_too_small_on_average(fmt):
    """The mean of the results' relative errors, over 2^20 of them behind one block of 128 positive values.

    Each result is rounded to float16: an error of mean 0 and at most 2^-11, so the mean of all of them has a standard
    deviation below 2^-11 / sqrt(3) / 2^10 < 2^-21.7.  A block's 16 products add to float32 sums that lose at most 2^-23 of
    their value each time, half of it on average: below 2^-20 in all.  A second part of a weight rounded to the nearest is off
    by 2^-16 at most and by nothing on average; one that is cut off is too small by 2^-17.1 on average (weights 2^-6 to 1).
    Four standard deviations and the sums: 2^-20 + 2^-19.7 < 2^-18.8."""
    from epure import paged
    B, H, hd = 1024, 8, 128
    pages, starts, prefix, seq, lengths, _ = _case([(128, [0] * B)], 1, hd, 64, fmt, torch.float16)
    g = _gen(21)
    at, pos = torch.zeros(128, dtype=torch.int32, device=DEV), torch.arange(128, device=DEV)
    k = torch.randn(128, 1, hd, generator=g, device=DEV).half()
    v = (0.5 + 0.5 * torch.rand(128, 1, hd, generator=g, device=DEV)).half()
    paged.write(pages, k, v, at, pos)
    k, v = (x[:, 0].double() for x in paged.read(pages, at, pos, torch.float32))
    q = torch.randn(B, H, hd, generator=g, device=DEV).half()
    out = paged.attend_shared(pages, q, torch.tensor(lengths, device=DEV), starts, prefix, seq=seq, always=True)
    want = torch.softmax(q.double() @ k.T / math.sqrt(hd), -1) @ v
    mean = float(((out.double() - want) / want).mean())
    assert abs(mean) <= 2.0 ** -18.8, math.log2(abs(mean))


def test_many_groups():
    """More tiles than a warp looks at together, of two to five rows, with empty groups and groups of one row between."""
    groups = [(37 + 61 * (i % 17), [[3, 0], [1, 9, -1, 4], [5], [], [2, 2, 7], [0, 1, 2, 3, 4]][i % 6]) for i in range(90)]
    for fmt in ("same", "int8"):
        case = _case(groups, 2, 64, 16, fmt, torch.bfloat16)
        _check(case, _q(case, 8, 64, torch.bfloat16))


@pytest.mark.parametrize("fmt,hd", [("same", 16), ("int8", 16), ("same", 48)])
def test_more_groups_than_the_plan_holds(fmt, hd):
    """More groups and tiles than the plan's threads and shared memory hold (512 each), of small heads."""
    groups = [(5 + 13 * (i % 29), [1, 2] if i % 7 else [1, 2, 3]) for i in range(1100)]
    case = _case(groups, 1, hd, 8, fmt, torch.bfloat16, same=True)
    _check(case, _q(case, 2, hd, torch.bfloat16))


def test_layouts():
    """Rows of a projection, unaligned rows, heads by rows, an output that is given, the default sequences."""
    from epure import paged
    case = _case([(9000, [7, 0, 30, 12] * 6)], 2, 128, 64, "same", torch.bfloat16)
    pages, starts, prefix, seq, lengths, _ = case
    n = torch.tensor(lengths, device=DEV)
    wide = torch.randn(24, 20, 128, generator=_gen(6), device=DEV).to(torch.bfloat16)
    q = wide[:, 2:10]
    want = paged.attend_shared(pages, q.contiguous(), n, starts, prefix, seq=seq, always=True)
    odd = torch.empty(24 * 8 * 128 + 2, dtype=q.dtype, device=DEV)[2:].view(24, 8, 128).copy_(q)
    odder = torch.empty(24 * 8 * 128 + 1, dtype=q.dtype, device=DEV)[1:].view(24, 8, 128).copy_(q)
    swap = torch.empty(8, 24, 128, dtype=q.dtype, device=DEV).transpose(0, 1).copy_(q)
    for x in (q, odd, odder, swap):
        assert torch.equal(paged.attend_shared(pages, x, n, starts, prefix, always=True), want)
    out = torch.empty_like(want)
    version = out._version
    assert paged.attend_shared(pages, q, n, starts, prefix, out=out, always=True) is out and torch.equal(out, want) and out._version > version


def test_captured_and_replayed():
    """One graph over lengths, groups and prefixes that change between replays, next to eager calls on another stream."""
    from epure import paged
    case = _case([(9000, [7, 0, 30, 12] * 6)], 2, 128, 64, "same", torch.bfloat16)
    pages, starts, prefix, seq, lengths, _ = case
    q, n = _q(case, 8, 128, torch.bfloat16), torch.tensor(lengths, device=DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        paged.attend_shared(pages, q, n, starts, prefix, seq=seq, always=True)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, lse = paged.attend_shared(pages, q, n, starts, prefix, seq=seq, return_lse=True, always=True)
    for change in (lambda: None, lambda: n.sub_(100), lambda: prefix.fill_(4321), lambda: n[5:9].zero_(),
                   lambda: starts.copy_(torch.tensor([2, 20], dtype=torch.int32)), lambda: prefix.fill_(0)):
        change()
        torch.cuda.synchronize()
        graph.replay()
        with torch.cuda.stream(side):
            want = paged.attend_shared(pages, q, n, starts, prefix, seq=seq, return_lse=True, always=True)
        torch.cuda.synchronize()
        assert torch.equal(out, want[0]) and torch.equal(lse, want[1])


def test_little_to_share_is_not_shared():
    """Batches that are not worth a plan give attention's own results, bit for bit."""
    from epure import paged
    case = _case([(300, [5, 6, 7]), (40, [1, 2])], 2, 64, 16, "same", torch.bfloat16)
    pages, starts, prefix, seq, lengths, _ = case
    q, n = _q(case, 8, 64, torch.bfloat16), torch.tensor(lengths, device=DEV)
    assert torch.equal(paged.attend_shared(pages, q, n, starts, prefix, seq=seq), paged.attend(pages, q, n, seq=seq))
    case = _case([(9000, [5] * 24)], 2, 128, 64, "same", torch.bfloat16)
    pages, starts, prefix, seq, lengths, _ = case
    q, n = _q(case, 8, 128, torch.bfloat16), torch.tensor(lengths, device=DEV)
    few = torch.tensor([0, 1], dtype=torch.int32, device=DEV)              # known on the device alone
    assert torch.equal(paged.attend_shared(pages, q, n, few, prefix, seq=seq, always=True), paged.attend(pages, q, n, seq=seq))


@pytest.mark.parametrize("rows,tokens,shares", [(24, 9000, False), (100, 9000, True), (3, 9000, False)])
def test_shares_where_it_is_reckoned_to_be_faster(rows, tokens, shares):
    """Told apart by tables that, against the rules, name zeros in all rows but the first."""
    from epure import paged
    case = _case([(tokens, [5] * rows)], 2, 128, 64, "same", torch.bfloat16, spare=1)
    pages, starts, prefix, seq, lengths, _ = case
    zero = torch.ones(pages.k.shape[0], dtype=torch.bool, device=DEV)
    zero[pages.table[pages.table >= 0].long()] = False
    zero = int(zero.nonzero()[0])
    pages.k[zero], pages.v[zero] = 0, 0
    pages.table[1:, :tokens // 64] = zero
    q, n = _q(case, 8, 128, torch.bfloat16), torch.tensor(lengths, device=DEV)
    alone = paged.attend(pages, q, n)
    together = paged.attend_shared(pages, q, n, starts, prefix, always=True)
    assert not torch.equal(alone, together)
    assert torch.equal(paged.attend_shared(pages, q, n, starts, prefix), together if shares else alone)


def test_refusals():
    from epure import paged
    case = _case([(300, [5, 6, 7])], 2, 64, 16, "same", torch.bfloat16)
    pages, starts, prefix, seq, lengths, _ = case
    q, n = _q(case, 4, 64, torch.bfloat16), torch.tensor(lengths, device=DEV)
    for bad in (dict(starts=starts.long()), dict(starts=starts[:1]), dict(prefix=prefix.int()), dict(prefix=prefix.view(1, 1)),
                dict(starts=starts.cpu()), dict(prefix=prefix.cpu()), dict(lengths=n.int()), dict(seq=seq.long()),
                dict(out=torch.empty(3, 4, 32, device=DEV)), dict(out=torch.empty(4, 3, 64, dtype=q.dtype, device=DEV).transpose(0, 1))):
        kw = {**dict(lengths=n, starts=starts, prefix=prefix, seq=seq), **bad}
        with pytest.raises(RuntimeError, match="must be"):
            paged.attend_shared(pages, q, **kw, always=True)
    with pytest.raises(TypeError, match="queries"):
        paged.attend_shared(pages, q.float(), n, starts, prefix, always=True)
    with pytest.raises(RuntimeError, match="query heads"):
        paged.attend_shared(pages, q[:, :3], n, starts, prefix, always=True)
    with pytest.raises(RuntimeError, match="gradient"):
        paged.attend_shared(pages, q.clone().requires_grad_(), n, starts, prefix, always=True)
    empty = paged.attend_shared(pages, q[:0], n[:0], starts[:1], prefix[:0], return_lse=True, always=True)
    assert empty[0].shape == (0, 4, 64) and empty[1].shape == (0, 4)


_CHILD = r"""
import sys, torch
sys.path.insert(0, sys.argv[1])
from epure import _native, paged
dev, kind = "cuda:0", sys.argv[2]
g = torch.Generator(device=dev).manual_seed(0)
k = torch.randn(200, 2, 64, 128, device=dev, generator=g).to(torch.bfloat16)
table = torch.arange(160, dtype=torch.int32, device=dev).repeat(24, 1)
pages = paged.KVPages(k, k.flip(0), table)
q = torch.randn(24, 8, 128, device=dev, generator=g).to(torch.bfloat16)
t = lambda *v: torch.tensor(v, device=dev)
n = torch.full((24,), 10000, device=dev)
starts, prefix = t(0, 24).int(), t(9000)
assert _native.device_error() == 0
want = paged.attend(pages, q, n)
if kind == "starts":
    for bad in (t(0, 25).int(), t(-1, 24).int(), t(20, 4).int()):
        assert torch.equal(paged.attend_shared(pages, q, n, bad, prefix, always=True), want)
elif kind == "prefix":
    for bad in (-1, 10241):
        assert torch.equal(paged.attend_shared(pages, q, n, starts, t(bad), always=True), want)
elif kind == "length":                                 # bad rows are empty, the others go on
    n[3], n[7] = -5, 10241
    out = paged.attend_shared(pages, q, n, starts, prefix, always=True)
    keep = torch.ones(24, dtype=torch.bool, device=dev)
    keep[3] = keep[7] = False
    assert not out[~keep].any()
    assert float((out[keep].double() - want[keep].double()).abs().max()) <= 2 ** -7 * float(want.abs().max())
elif kind == "page":                                   # the tokens of a bad page are left out
    table[:, 5] = 200
    table[:, 6] = -3
    out, lse = paged.attend_shared(pages, q, n, starts, prefix, return_lse=True, always=True)
    a, la = paged.attend(pages, q, n, return_lse=True)
    assert float((out.double() - a.double()).abs().max()) <= 2 ** -7 * float(a.abs().max())
    assert float((lse - la).abs().max()) <= 1e-4
elif kind == "seq":
    seq = torch.arange(24, dtype=torch.int32, device=dev)
    seq[0], seq[9] = -1, 24
    out = paged.attend_shared(pages, q, n, starts, prefix, seq=seq, always=True)
    assert not out[[0, 9]].any() and out[1:9].any(-1).all()
torch.cuda.synchronize()
print("FLAG", _native.device_error())
"""


@pytest.mark.parametrize("kind,flag", [("starts", 16), ("prefix", 16), ("length", 16), ("page", 32), ("seq", 16)])
def test_bad_groups_lengths_and_pages_are_reported(kind, flag):
    """Skipped and reported by epq_device_error (in a child process: the flag stays set)."""
    r = subprocess.run([sys.executable, "-c", _CHILD, PKG, kind], capture_output=True, text=True, timeout=300,
                       env=dict(os.environ))
    assert r.returncode == 0, r.stderr[-2000:]
    assert f"FLAG {flag}" in r.stdout


_SMALL = r"""
import sys, torch
sys.path.insert(0, sys.argv[1])
from epure import _native, paged
dev, kind = "cuda:0", sys.argv[2]
t = lambda *v: torch.tensor(v, device=dev)
ps, always = (7, True) if kind == "pages" else (16, False)
k = torch.randn(12, 2, ps, 64, device=dev).to(torch.bfloat16)
pages = paged.KVPages(k, k.flip(0), torch.arange(12, dtype=torch.int32, device=dev).view(3, 4))
q = torch.randn(3, 4, 64, device=dev).to(torch.bfloat16)
n = t(20, 4, 28)
want = paged.attend(pages, q, n)
call = lambda starts, prefix: paged.attend_shared(pages, q, n, starts, prefix, always=always)
groups = 700 if kind == "last" else 1
good = t(*[0] * groups, 3).int(), t(*[4] * groups)
assert torch.equal(call(*good), want)
assert torch.equal(call(t(0).int(), t(0)[:0]), want)
assert _native.device_error() == 0
if kind == "prefix":
    bad = t(0, 3).int(), t(4 * ps + 1)
elif kind == "negative":
    bad = t(0, 3).int(), t(-1)
elif kind == "descending":
    bad = t(2, 1).int(), t(4)
elif kind == "last":
    bad = t(*[0] * 700, 4).int(), good[1]
else:
    bad = t(0, 4).int(), t(4)
assert torch.equal(call(*bad), want)
torch.cuda.synchronize()
print("FLAG", _native.device_error())
"""


@pytest.mark.parametrize("kind", ["starts", "prefix", "negative", "descending", "last", "pages"])
def test_bad_groups_are_reported_where_nothing_is_shared(kind):
    """Also where a batch is read row by row from the start: too little to share, or pages that cannot be (in a child process:
    the flag stays set)."""
    r = subprocess.run([sys.executable, "-c", _SMALL, PKG, kind], capture_output=True, text=True, timeout=300,
                       env=dict(os.environ))
    assert r.returncode == 0, r.stderr[-2000:]
    assert "FLAG 16" in r.stdout
