"""The paged cache (epq_paged_write / epq_paged_read) and its attention (epq_paged_attend) against plain
implementations in 64 bits."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
UNIT = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}   # unit roundoff
TOP = {"int8": 127.0, "fp8": 448.0}


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from epure import _native
    _native.load_library()
    yield
    assert _native.device_error() == 0


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _pages(lengths, kv, hd, ps, fmt, dtype, seed=0, junk=float("nan"), spare=2):
    """A cache whose pages lie in a random order; every slot that is no token holds `junk`."""
    from epure.paged import FORMATS, KVPages
    g = _gen(seed)
    need = [-(-n // ps) for n in lengths]
    total = sum(need) + spare
    order = torch.randperm(total, generator=g, device=DEV).int().cpu()
    table = torch.full((len(lengths), max(1, max(need))), -1, dtype=torch.int32)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n]
        at += n
    store = FORMATS[fmt] or dtype
    shape = (total, kv, ps, hd)
    if fmt == "same":
        return KVPages(torch.full(shape, junk, dtype=store, device=DEV), torch.full(shape, junk, dtype=store, device=DEV),
                       table.to(DEV))
    codes = [torch.full(shape, 0x7f, dtype=torch.int8, device=DEV).view(store) for _ in range(2)]   # NaN as e4m3
    scales = [torch.full(shape[:3], junk, device=DEV) for _ in range(2)]
    return KVPages(*codes, table.to(DEV), *scales)


def _tokens(lengths):
    seq = torch.cat([torch.full((n,), i, dtype=torch.int32) for i, n in enumerate(lengths)]).to(DEV)
    pos = torch.cat([torch.arange(n) for n in lengths]).to(DEV)
    return seq, pos


def _stored(x, fmt):
    """(values the cache stands for in float32, scales) of rows x, by the documented float32 steps."""
    f = x.float()
    if fmt == "same":
        return f, None
    a = f.abs().amax(-1, keepdim=True)
    inv = torch.where(a > 0, torch.full_like(a, TOP[fmt]) / a, torch.zeros_like(a))
    c = f * inv
    c = c.round() if fmt == "int8" else c.to(torch.float8_e4m3fn).float()
    s = a * (1.0 / TOP[fmt])
    return c * s, s


# -- write and read ----------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("fmt", ["same", "int8", "fp8"])
@pytest.mark.parametrize("lengths,kv,hd,ps", [([1], 8, 128, 16), ([5, 0, 33], 2, 64, 16), ([70, 3], 3, 80, 7),
                                              ([9, 12], 1, 256, 1), ([300], 4, 16, 64)])
def test_write_then_read(dtype, fmt, lengths, kv, hd, ps):
    """Reading gives code * scale of the documented float32 steps bit for bit, and is as near to the row as the
    format allows: half a step of int8 (scale / 2), 2^-4 of the value (or half of e4m3's smallest step, 2^-10
    scales) for fp8, plus the float32 roundings and the one to dtype."""
    from epure import paged
    pages = _pages(lengths, kv, hd, ps, fmt, dtype)
    seq, pos = _tokens(lengths)
    g = _gen(1)
    kvs = torch.randn(len(pos), 2 * kv, hd, generator=g, device=DEV) * torch.rand(len(pos), 2 * kv, 1, generator=g,
                                                                                  device=DEV).exp2()
    kvs = kvs.to(dtype)
    k, v = kvs[:, :kv], kvs[:, kv:]                    # views with a row stride of 2 kv heads
    k[0, 0] = 0                                        # a row of zeros
    order = torch.randperm(len(pos), generator=g, device=DEV)
    assert paged.write(pages, k[order], v[order], seq[order], pos[order]) is None
    got = paged.read(pages, seq, pos, dtype)
    for x, y in zip((k, v), got):
        want, scale = _stored(x, fmt)
        assert torch.equal(y, want.to(dtype))
        err = (y.double() - x.double()).abs()
        if fmt == "same":
            assert not err.any()
        else:
            step = scale.double() * 0.5 if fmt == "int8" else \
                torch.maximum(x.double().abs() * 2.0 ** -4, scale.double() * 2.0 ** -10)
            assert bool((err <= step * (1 + 2.0 ** -20) + 2 * UNIT[dtype] * x.double().abs() + 1e-30 +
                         scale.double() * 2.0 ** -16).all())
    again = paged.read(pages, seq.flip(0), pos.flip(0), dtype)
    assert torch.equal(again[0].flip(0), got[0])
    wide = paged.read(pages, seq, pos, torch.float32) if fmt != "same" else None
    if wide is not None:
        assert torch.equal(wide[0], _stored(k, fmt)[0])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("heads,kv,hd,r", [(8, 2, 64, 64), (4, 4, 128, 128), (6, 2, 80, 32), (2, 1, 96, 50), (3, 1, 256, 256)])
def test_write_rotates_as_rope(dtype, interleaved, heads, kv, hd, r):
    """The fused rotation of q and k equals epq_rope's results bit for bit; v is not rotated."""
    from epure import paged, rotary
    lengths = [40, 3]
    pages = _pages(lengths, kv, hd, 16, "same", dtype)
    seq, pos = _tokens(lengths)
    qkv = torch.randn(len(pos), heads + 2 * kv, hd, generator=_gen(2), device=DEV).to(dtype)
    q, k, v = qkv[:, :heads], qkv[:, heads:heads + kv], qkv[:, heads + kv:]
    cos, sin = rotary.rope_tables(r, 64, DEV)
    want = rotary.rope(q, k, pos, cos, sin, interleaved=interleaved)
    got_q = paged.write(pages, k, v, seq, pos, q=q, cos=cos, sin=sin, interleaved=interleaved)
    rk, rv = paged.read(pages, seq, pos)
    assert torch.equal(got_q, want[0]) and torch.equal(rk, want[1]) and torch.equal(rv, v)
    if r % 16 == 0 or interleaved:
        q2 = q.contiguous()
        paged.write(pages, k, v, seq, pos, q=q2, q_out=q2, cos=cos, sin=sin, interleaved=interleaved)
        assert torch.equal(q2, want[0])


@pytest.mark.parametrize("r", [0, 64, 20])
def test_write_norms_heads(r):
    """RMSNorm of q and k before the rotation: one float32 norm of relative error below hd 2^-23, one rounding to
    the type, then the rotation of the rounded values (another rounding); values of at most sqrt(hd)."""
    from epure import paged, rotary
    H, KV, hd = 4, 2, 64
    pages = _pages([30], KV, hd, 16, "same", torch.bfloat16)
    seq, pos = _tokens([30])
    x = torch.randn(30, H + 2 * KV, hd, generator=_gen(4), device=DEV).to(torch.bfloat16) * 3
    q, k, v = x[:, :H], x[:, H:H + KV], x[:, H + KV:]
    cos, sin = rotary.rope_tables(r, 64, DEV) if r else (None, None)
    got_q = paged.write(pages, k, v, seq, pos, q=q, cos=cos, sin=sin, qk_norm=True, eps=1e-5)
    got_k, got_v = paged.read(pages, seq, pos)
    assert torch.equal(got_v, v)
    for t, got in ((q, got_q), (k, got_k)):
        d = t.double()
        n = d / (d.square().mean(-1, keepdim=True) + 1e-5).sqrt()
        y = n.clone()
        bound = 1.5 * 2.0 ** -8 * n.abs()              # the norm's rounding (and its float32 error)
        if r:
            c, s = cos.double()[pos][:, None], sin.double()[pos][:, None]
            a, b = n[..., :r // 2], n[..., r // 2:r]
            y[..., :r // 2], y[..., r // 2:r] = a * c - b * s, b * c + a * s
            ba, bb = bound[..., :r // 2].clone(), bound[..., r // 2:r].clone()
            bound[..., :r // 2] = bound[..., r // 2:r] = ba + bb
        assert bool(((got.double() - y).abs() <= bound + 2.0 ** -8 * y.abs() + 1e-6).all())


def test_padding_rows_and_other_sequences_stay():
    from epure import paged
    pages = _pages([20, 20], 2, 64, 16, "int8", torch.bfloat16, junk=1.0)
    before = [t.clone() for t in (pages.k, pages.v, pages.k_scale, pages.v_scale)]
    x = torch.randn(3, 2, 64, device=DEV).to(torch.bfloat16)
    q = torch.randn(3, 4, 64, device=DEV).to(torch.bfloat16)
    seq = torch.tensor([0, 7, 1], dtype=torch.int32, device=DEV)
    pos = torch.tensor([3, -1, -5], device=DEV)
    got = paged.write(pages, x, x, seq, pos, q=q)
    assert torch.equal(got[0], q[0]) and not got[1:].any()
    k, v = paged.read(pages, seq, pos)
    assert not k[1:].any() and not v[1:].any() and k[0].any()
    page = int(pages.table[0, 0])
    for t, b in zip((pages.k, pages.v, pages.k_scale, pages.v_scale), before):
        assert not torch.equal(t[page, :, 3], b[page, :, 3])
        t[page, :, 3] = b[page, :, 3]
        assert torch.equal(t, b)


def test_not_finite_tiny_and_large_rows():
    """A row with an infinity or NaN reads back as NaN; the others keep their precision at every magnitude."""
    from epure import paged
    for fmt in ("int8", "fp8"):
        pages = _pages([8], 1, 64, 16, fmt, torch.float32)
        seq, pos = _tokens([8])
        x = torch.randn(8, 1, 64, generator=_gen(5), device=DEV)
        for i, m in enumerate((1.0, 1e-30, 1e-38, 1e-42, 1e37)):
            x[i] *= m
        x[5, 0, 9] = float("inf")
        x[6, 0, 1] = float("nan")
        paged.write(pages, x, x, seq, pos)
        k, _ = paged.read(pages, seq, pos, torch.float32)
        assert torch.isnan(k[5:7]).all() and torch.isfinite(k[:5]).all() and torch.isfinite(k[7]).all()
        for i in (0, 1, 2, 3, 4, 7):
            a = x[i].double().abs().max()
            # half a step of the largest value; where float32 itself is coarse (subnormal scales) its step times the code
            step = a / 254 if fmt == "int8" else a / 16
            assert float((k[i].double() - x[i].double()).abs().max()) <= float(step * 1.001 + 2.0 ** -149 * TOP[fmt] * 1.5)


@pytest.mark.parametrize("fmt", ["same", "int8"])
def test_pools_side_by_side_and_a_wider_table(fmt):
    """Keys and values as the two halves of one pool's pages (a page stride of two), and a table that is a part of
    a wider one."""
    from epure import paged
    lengths = [37, 90]
    plain = _pages(lengths, 2, 64, 16, fmt, torch.bfloat16)
    both = torch.stack((plain.k.view(torch.int8), plain.v.view(torch.int8)), 1).view(plain.k.dtype)
    scales = (None, None) if fmt == "same" else torch.stack((plain.k_scale, plain.v_scale), 1).unbind(1)
    wide = torch.full((2, 40), 10 ** 6, dtype=torch.int32, device=DEV)
    wide[:, 3:3 + plain.table.shape[1]] = plain.table
    pages = paged.KVPages(both[:, 0], both[:, 1], wide[:, 3:3 + plain.table.shape[1]], *scales)
    assert pages.k.stride(0) == 2 * 2 * 16 * 64
    got = _fill(pages, lengths, torch.bfloat16)
    want = _fill(plain, lengths, torch.bfloat16)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    q = torch.randn(2, 8, 64, generator=_gen(23), device=DEV).to(torch.bfloat16)
    n = torch.tensor(lengths, device=DEV)
    assert torch.equal(paged.attend(pages, q, n), paged.attend(plain, q, n))
    _check(pages, q, lengths, *got)


def test_unaligned_rows():
    from epure import paged
    pages = _pages([6], 2, 32, 16, "same", torch.bfloat16)
    seq, pos = _tokens([6])
    flat = torch.randn(6 * 2 * 32 + 1, device=DEV).to(torch.bfloat16)
    x = flat[1:].view(6, 2, 32)
    paged.write(pages, x, x, seq, pos, q=x, q_out=torch.empty(6 * 64 + 1, dtype=x.dtype, device=DEV)[1:].view(6, 2, 32))
    assert torch.equal(paged.read(pages, seq, pos)[1], x)


# -- attention ---------------------------------------------------------------------------------------------------

def _fill(pages, lengths, dtype, seed=1, scale_range=0.0):
    """Writes random tokens; the dequantised keys and values [tokens, kv, hd] in 64 bits."""
    from epure import paged
    g = _gen(seed)
    seq, pos = _tokens(lengths)
    shape = (len(pos), pages.k.shape[1], pages.k.shape[3])
    k = torch.randn(shape, generator=g, device=DEV)
    v = torch.randn(shape, generator=g, device=DEV)
    if scale_range:
        v *= torch.exp2(scale_range * (2 * torch.rand(shape[:2], generator=g, device=DEV) - 1))[..., None]
    k, v = k.to(dtype), v.to(dtype)
    if len(pos):
        paged.write(pages, k, v, seq, pos)
        if pages.k_scale is not None:
            k, v = paged.read(pages, seq, pos, torch.float32)
    return k.double(), v.double()


def _reference(q, k, v, lengths, window, scale):
    """(out, lse, weighted |v|, bound on a score's error) in 64 bits."""
    B, H, hd = q.shape
    kv = k.shape[1]
    out = torch.zeros(B, H, hd, dtype=torch.float64, device=DEV)
    lse = torch.full((B, H), -math.inf, dtype=torch.float64, device=DEV)
    mag, err = torch.zeros_like(out), torch.zeros_like(lse)
    at = 0
    for b, n in enumerate(lengths):
        lo = max(0, n - window) if window else 0
        kk, vv = k[at + lo:at + n], v[at + lo:at + n]
        at += n
        if n == 0:
            continue
        for h in range(H):
            j = h // (H // kv)
            z = kk[:, j] @ q[b, h].double() * scale
            p = torch.softmax(z, 0)
            out[b, h], mag[b, h] = p @ vv[:, j], p @ vv[:, j].abs()
            lse[b, h] = torch.logsumexp(z, 0)
            # hd products summed in float32, and the scaled score's own rounding
            err[b, h] = 2.0 ** -23 * (hd * float((kk[:, j].abs() @ q[b, h].double().abs()).max()) * scale +
                                      4 * float(z.abs().max()))
    return out, lse, mag, err


def _check(pages, q, lengths, k, v, window=0, seq=None, scale=None, **kw):
    """Bounds: a weight is rounded once (unit roundoff of the tensor-core type: q's for 16-bit caches, f16 for
    8-bit ones; f16 weights below 2^-14 round by up to 2^-25 of the largest contribution each), carries its score's error
    twice (numerator and sum) and about 2^-18 of exp2, log2 and the sums; the result is rounded once more."""
    from epure import paged
    sc = 1 / math.sqrt(q.shape[-1]) if scale is None else scale
    out, lse = paged.attend(pages, q, torch.tensor(lengths, device=DEV), seq=seq, window=window, scale=scale,
                            return_lse=True, **kw)
    want, want_lse, mag, err = _reference(q, k, v, lengths, window, sc)
    p_unit = UNIT[torch.float16] if pages.k_scale is not None else UNIT[q.dtype]
    small = 2.0 ** -25 * max(lengths) * float(v.abs().max()) if p_unit == 2.0 ** -11 and v.numel() else 0.0
    bound = UNIT[q.dtype] * want.abs() + (p_unit + 2 * err[..., None] + 2.0 ** -18) * 1.01 * mag + small + 2.0 ** -25
    off = (out.double() - want).abs()
    assert bool((off <= bound).all()), (float((off / bound.clamp(min=1e-30)).max()), float(off.max()))
    empty = torch.isinf(want_lse)
    assert torch.equal(torch.isneginf(lse), empty) and not out[empty].any()
    off = (lse.double() - want_lse)[~empty].abs()
    assert bool((off <= err[~empty] + 2.0 ** -20 * (1 + want_lse[~empty].abs())).all()), float(off.max())
    return out, lse


LENGTHS = [0, 1, 15, 16, 17, 63, 64, 65, 333, 0, 1000]


@pytest.mark.parametrize("fmt", ["same", "int8", "fp8"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("heads,kv,hd,ps", [(32, 8, 128, 16), (8, 2, 64, 64), (4, 4, 128, 48), (12, 4, 80, 7),
                                            (28, 4, 128, 16), (16, 1, 64, 1), (40, 2, 64, 24), (6, 2, 256, 16),
                                            (24, 2, 256, 5), (3, 3, 16, 16), (5, 1, 48, 128), (9, 1, 112, 32)])
def test_attend(fmt, dtype, heads, kv, hd, ps):
    pages = _pages(LENGTHS, kv, hd, ps, fmt, dtype)
    k, v = _fill(pages, LENGTHS, dtype)
    q = (torch.randn(len(LENGTHS), heads, hd, generator=_gen(7), device=DEV) * 2).to(dtype)
    one, lse = _check(pages, q, LENGTHS, k, v)
    from epure import paged
    two = paged.attend(pages, q, torch.tensor(LENGTHS, device=DEV))
    assert torch.equal(one, two)                       # the joining order is fixed


@pytest.mark.parametrize("fmt", ["same", "int8"])
@pytest.mark.parametrize("window", [1, 15, 16, 17, 100, 5000])
def test_window(fmt, window):
    pages = _pages(LENGTHS, 2, 64, 24, fmt, torch.bfloat16)
    k, v = _fill(pages, LENGTHS, torch.bfloat16)
    q = torch.randn(len(LENGTHS), 8, 64, generator=_gen(8), device=DEV).to(torch.bfloat16)
    _check(pages, q, LENGTHS, k, v, window=window)


@pytest.mark.parametrize("fmt", ["same", "int8", "fp8"])
def test_one_long_sequence_and_many_short(fmt):
    """A unit cut over many CTAs, and more sequences than a CTA's threads."""
    lengths = [20011]
    pages = _pages(lengths, 2, 128, 64, fmt, torch.bfloat16)
    k, v = _fill(pages, lengths, torch.bfloat16)
    q = torch.randn(1, 16, 128, generator=_gen(9), device=DEV).to(torch.bfloat16)
    _check(pages, q, lengths, k, v)
    lengths = [(i * 37) % 61 if i % 3 else 0 for i in range(400)]
    pages = _pages(lengths, 1, 64, 16, fmt, torch.bfloat16)
    k, v = _fill(pages, lengths, torch.bfloat16)
    q = torch.randn(400, 2, 64, generator=_gen(10), device=DEV).to(torch.bfloat16)
    _check(pages, q, lengths, k, v)
    _check(pages, q[:, :, :], [0] * 400, k[:0], v[:0])


def test_uneven_scores_and_scales():
    """Peaked scores whose maximum keeps rising along the sequence, and value rows whose scales differ by 2^24."""
    for fmt in ("same", "int8", "fp8"):
        lengths = [700, 300]
        pages = _pages(lengths, 2, 64, 16, fmt, torch.bfloat16)
        k, v = _fill(pages, lengths, torch.bfloat16, scale_range=12.0)
        q = torch.randn(2, 8, 64, generator=_gen(11), device=DEV).to(torch.bfloat16)
        _check(pages, q * 12, lengths, k, v)
        _check(pages, q * 1e-4, lengths, k, v)
        _check(pages, q, lengths, k, v, scale=2.5)
        _check(pages, q, lengths, k, v, scale=0.0)


def test_small_and_large_queries_over_8_bit_caches():
    """q outside f16's range is scaled by a power of two, not clipped."""
    lengths = [100]
    pages = _pages(lengths, 1, 64, 16, "int8", torch.bfloat16)
    k, v = _fill(pages, lengths, torch.bfloat16)
    q = torch.randn(1, 4, 64, generator=_gen(12), device=DEV)
    _check(pages, (q * 1e20).to(torch.bfloat16), lengths, k, v, scale=1e-20)
    _check(pages, (q * 1e-30).to(torch.bfloat16), lengths, k, v, scale=1e29)
    mixed = torch.cat((q[..., :32] * 1e6, q[..., 32:] * 1e-3), -1).to(torch.bfloat16)
    _check(pages, mixed, lengths, k, v, scale=1e-6)
    _check(pages, torch.zeros_like(q).to(torch.bfloat16), lengths, k, v)


def test_not_finite_values_stay_in_their_row():
    from epure import paged
    lengths = [40, 40, 40]
    for fmt in ("same", "int8"):
        pages = _pages(lengths, 1, 64, 16, fmt, torch.bfloat16)
        seq, pos = _tokens(lengths)
        k = torch.randn(120, 1, 64, generator=_gen(13), device=DEV).to(torch.bfloat16)
        v = torch.randn(120, 1, 64, generator=_gen(14), device=DEV).to(torch.bfloat16)
        v[50, 0, 5] = float("nan")                     # sequence 1
        k[90, 0, 5] = float("nan")                     # sequence 2
        paged.write(pages, k, v, seq, pos)
        q = torch.randn(3, 2, 64, generator=_gen(15), device=DEV).to(torch.bfloat16)
        out = paged.attend(pages, q, torch.tensor(lengths, device=DEV))
        assert torch.isfinite(out[0]).all() and torch.isnan(out[2]).all()
        bad = torch.isnan(out[1])
        assert bad[:, 5].all() and (fmt != "same" or int(bad.sum()) == 2)


def test_scores_of_minus_infinity():
    """Keys of -inf leave weight 0; a row whose every score is -inf counts as empty."""
    from epure import paged
    pages = _pages([20, 20], 1, 16, 16, "same", torch.float16)
    seq, pos = _tokens([20, 20])
    k = torch.randn(40, 1, 16, generator=_gen(16), device=DEV).half().abs()
    v = torch.randn(40, 1, 16, generator=_gen(17), device=DEV).half()
    k[3, 0, 0] = k[17, 0, 0] = float("-inf")
    k[20:, 0, 0] = float("-inf")
    paged.write(pages, k, v, seq, pos)
    q = torch.ones(2, 1, 16, dtype=torch.float16, device=DEV)
    out, lse = paged.attend(pages, q, torch.tensor([20, 20], device=DEV), return_lse=True)
    z = k[:20, 0].double().sum(-1) / 4
    p = torch.softmax(z, 0)
    assert float((out[0, 0].double() - p @ v[:20, 0].double()).abs().max()) <= 2.0 ** -9
    assert not out[1].any() and float(lse[1, 0]) == -math.inf


def test_subset_of_sequences_strided_queries_and_out():
    from epure import paged
    lengths = [100, 37, 5, 260]
    pages = _pages(lengths, 2, 64, 16, "fp8", torch.bfloat16)
    _fill(pages, lengths, torch.bfloat16)
    full = torch.randn(4, 12, 64, generator=_gen(18), device=DEV).to(torch.bfloat16)
    q = full[:, :8]                                    # the q part of a fused projection
    want = paged.attend(pages, q.contiguous(), torch.tensor(lengths, device=DEV))
    assert torch.equal(paged.attend(pages, q, torch.tensor(lengths, device=DEV)), want)
    pick = torch.tensor([3, 1], dtype=torch.int32, device=DEV)
    out = torch.empty(2, 8, 64, dtype=torch.bfloat16, device=DEV)
    got = paged.attend(pages, q[[3, 1]], torch.tensor([260, 37], device=DEV), seq=pick, out=out)
    assert got is out and torch.equal(got[1], want[1])
    assert float((got[0].float() - want[3].float()).abs().max()) <= 2.0 ** -7 * float(want[3].abs().max())
    odd = torch.empty(4 * 8 * 64 + 1, dtype=torch.bfloat16, device=DEV)[1:].view(4, 8, 64)
    odd.copy_(q)
    assert torch.equal(paged.attend(pages, odd, torch.tensor(lengths, device=DEV)), want)
    assert paged.attend(pages, q[:0], torch.tensor([], dtype=torch.long, device=DEV)).shape == (0, 8, 64)


def test_shared_pages_and_joined_results():
    """Two sequences may share pages; lse joins results over disjoint tokens."""
    from epure import paged
    pages = _pages([64, 64], 1, 64, 16, "same", torch.bfloat16)
    pages.table[1, :2] = pages.table[0, :2]
    seq, pos = _tokens([64, 64])
    x = torch.randn(128, 2, 64, generator=_gen(19), device=DEV).to(torch.bfloat16)
    keep = (seq == 0) | (pos >= 32)
    paged.write(pages, x[keep, :1], x[keep, 1:], seq[keep], pos[keep])
    q = torch.randn(1, 4, 64, generator=_gen(20), device=DEV).to(torch.bfloat16).expand(2, 4, 64)
    a, la = paged.attend(pages, q, torch.tensor([32, 32], device=DEV), return_lse=True)
    assert torch.equal(a[0], a[1]) and torch.equal(la[0], la[1])
    whole, lw = paged.attend(pages, q[:1], torch.tensor([64], device=DEV), return_lse=True)
    tail, lt = paged.attend(pages, q[:1], torch.tensor([64], device=DEV), window=32, return_lse=True)
    wa, wt = torch.exp(la[0] - lw[0]), torch.exp(lt[0] - lw[0])
    joined = wa[:, None] * a[0].float() + wt[:, None] * tail[0].float()
    assert float((joined - whole[0].float()).abs().max()) <= 2.0 ** -6
    assert float((torch.logaddexp(la[0], lt[0]) - lw[0]).abs().max()) <= 2.0 ** -18


@pytest.mark.parametrize("fmt", ["same", "int8"])
def test_offsets_past_32_bits(fmt):
    """Pages that lie beyond 2^31 values and 2^32 bytes of the pool."""
    from epure import paged
    kv, ps, hd = 8, 64, 128
    count = (2 ** 31 if fmt == "same" else 2 ** 32) // (kv * ps * hd) + 8
    store = torch.bfloat16 if fmt == "same" else torch.int8
    k, v = (torch.empty(count, kv, ps, hd, dtype=store, device=DEV) for _ in range(2))
    scales = (None, None) if fmt == "same" else tuple(torch.empty(count, kv, ps, device=DEV) for _ in range(2))
    table = torch.tensor([[count - 1, 0, count - 3]], dtype=torch.int32, device=DEV)
    pages = paged.KVPages(k, v, table, *scales)
    lengths = [150]
    kk, vv = _fill(pages, lengths, torch.bfloat16)
    q = torch.randn(1, 16, hd, generator=_gen(21), device=DEV).to(torch.bfloat16)
    _check(pages, q, lengths, kk, vv)


def test_side_stream_and_graph():
    """Calls on a stream of their own, and a captured step that replays at new positions and lengths."""
    from epure import paged, rotary
    H, KV, hd = 8, 2, 64
    pages = _pages([200, 200], KV, hd, 16, "int8", torch.bfloat16)
    _fill(pages, [200, 200], torch.bfloat16)
    cos, sin = rotary.rope_tables(hd, 256, DEV)
    seq = torch.arange(2, dtype=torch.int32, device=DEV)
    pos = torch.tensor([10, 20], device=DEV)
    x = torch.randn(2, H + 2 * KV, hd, generator=_gen(22), device=DEV).to(torch.bfloat16)

    def step():
        q = paged.write(pages, x[:, H:H + KV], x[:, H + KV:], seq, pos, q=x[:, :H], cos=cos, sin=sin)
        return paged.attend(pages, q, pos + 1)

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        aside = step()
    torch.cuda.current_stream().wait_stream(stream)
    assert torch.equal(aside, step())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for p in ([11, 21], [150, 0], [199, 199]):
        pos.copy_(torch.tensor(p))
        graph.replay()
        got = out.clone()
        assert torch.equal(got, step())


def test_refusals():
    from epure import paged
    pages = _pages([20], 2, 64, 16, "same", torch.bfloat16)
    q8 = _pages([20], 2, 64, 16, "int8", torch.bfloat16)
    x = torch.zeros(1, 2, 64, dtype=torch.bfloat16, device=DEV)
    q = torch.zeros(1, 4, 64, dtype=torch.bfloat16, device=DEV)
    seq, pos, n = torch.zeros(1, dtype=torch.int32, device=DEV), torch.zeros(1, dtype=torch.long, device=DEV), \
        torch.ones(1, dtype=torch.long, device=DEV)
    with pytest.raises(RuntimeError, match="rows of"):
        paged.write(pages, x.half(), x.half(), seq, pos)
    with pytest.raises(RuntimeError, match="expected"):
        paged.write(pages, q, q, seq, pos)
    with pytest.raises(RuntimeError, match="seq"):
        paged.write(pages, x, x, seq.long(), pos)
    with pytest.raises(RuntimeError, match="k_scale"):
        paged.write(q8._replace(k_scale=None), x, x, seq, pos)
    with pytest.raises(RuntimeError, match="no scales"):
        paged.write(pages._replace(k_scale=q8.k_scale), x, x, seq, pos)
    with pytest.raises(RuntimeError, match="contiguous"):
        paged.read(pages._replace(k=pages.k.transpose(1, 2), v=pages.v.transpose(1, 2)), seq, pos)
    with pytest.raises(RuntimeError, match="read as"):
        paged.read(pages, seq, pos, torch.float16)
    with pytest.raises(TypeError, match="float16 or bfloat16"):
        paged.attend(q8, q.float(), n)
    with pytest.raises(RuntimeError, match="queries of"):
        paged.attend(pages, q.half(), n)
    with pytest.raises(RuntimeError, match="query heads"):
        paged.attend(pages, torch.zeros(1, 5, 64, dtype=torch.bfloat16, device=DEV), n)
    with pytest.raises(RuntimeError, match="lengths"):
        paged.attend(pages, q, n.int())
    with pytest.raises(RuntimeError, match="table of 1"):
        paged.attend(pages, q.expand(2, 4, 64), n.expand(2).contiguous())
    with pytest.raises(RuntimeError, match="bad arguments"):
        paged.attend(pages, q, n, window=-1)
    with pytest.raises(RuntimeError, match="out must"):
        paged.attend(pages, q, n, out=torch.zeros(1, 4, 32, dtype=torch.bfloat16, device=DEV))
    with pytest.raises(RuntimeError, match="in place"):
        from epure import rotary
        cos, sin = rotary.rope_tables(20, 8, DEV)
        paged.write(pages, x, x, seq, pos, q=q, q_out=q, cos=cos, sin=sin)


_CHILD = r"""
import sys, torch
sys.path.insert(0, sys.argv[1])
from epure import _native, paged
dev, kind = "cuda:0", sys.argv[2]
k = torch.randn(4, 2, 16, 64, device=dev).to(torch.bfloat16)
pages = paged.KVPages(k, k.clone(), torch.tensor([[0, 1], [2, 9], [3, -1]], dtype=torch.int32, device=dev))
q = torch.randn(3, 4, 64, device=dev).to(torch.bfloat16)
x = torch.randn(1, 2, 64, device=dev).to(torch.bfloat16)
t = lambda *v: torch.tensor(v, device=dev)
assert _native.device_error() == 0
keep = pages.k.clone()
if kind == "length":
    out = paged.attend(pages, q, t(33, 16, -1))
    assert not out[0].any() and not out[2].any() and out[1].any()
elif kind == "page":
    out, lse = paged.attend(pages, q, t(32, 32, 32), return_lse=True)
    want = paged.attend(pages, q, t(32, 16, 16))
    assert torch.equal(out[0], want[0]) and torch.isfinite(out).all() and torch.isfinite(lse).all()
    assert float((out - want).abs().max()) <= 2 ** -7          # the bad page's tokens are left out
elif kind == "seq":
    out = paged.attend(pages, q, t(16, 16, 16), seq=t(0, 3, -1).int())
    assert out[0].any() and not out[1:].any()
elif kind == "write":
    paged.write(pages, x, x, t(1).int(), t(20))
    assert torch.equal(pages.k, keep)
elif kind == "write-pos":
    y = paged.write(pages, x, x, t(0).int(), t(32), q=q[:1])
    assert torch.equal(pages.k, keep) and not y.any()
elif kind == "read":
    a, b = paged.read(pages, t(2).int(), t(17))
    assert not a.any() and not b.any()
torch.cuda.synchronize()
print("FLAG", _native.device_error())
"""


@pytest.mark.parametrize("kind,flag", [("length", 16), ("page", 32), ("seq", 16), ("write", 32), ("write-pos", 16),
                                       ("read", 32)])
def test_bad_positions_and_pages_are_reported(kind, flag):
    """Skipped and reported by epq_device_error (in a child process: the flag stays set)."""
    import subprocess
    import sys
    from conftest import PKG
    r = subprocess.run([sys.executable, "-c", _CHILD, PKG, kind], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and f"FLAG {flag}" in r.stdout, r.stdout + r.stderr[-2000:]
