"""Verification of drafted tokens (epure.sampling.verify) against its definition in 64 bits, row by row."""
import math
import os
import subprocess
import sys

import pytest
import torch
from conftest import PKG

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from epure import _native
    _native.load_library()
    yield
    assert _native.device_error() == 0


def _expected(p, q, x, u):
    """The definition; cumulative sums on the CPU.  Also how near each drawn number came to a border, as a share of the sum."""
    B, K = x.shape
    out, count, near = [], [], []
    for b in range(B):
        n, toks = 0, x[b].tolist()
        while n < K and toks[n] >= 0:
            qx = 1.0 if q is None else float(q[b, n, toks[n]])
            if not float(u[b, n].double()) * qx < float(p[b, n, toks[n]]):
                break
            n += 1
        w = p[b, n].cpu().double()
        w = torch.where(w > 0, w, 0.0)
        if n < K and toks[n] >= 0:
            if q is None:
                less = w.clone()
                less[toks[n]] = 0
            else:
                less = p[b, n].cpu().double() - q[b, n].cpu().double()
                less = torch.where(less > 0, less, 0.0)
            w = less if bool(less.any()) else w
        c = torch.cumsum(w, 0)
        draw = float(u[b, K].double()) * float(c[-1])
        hit = torch.nonzero((c > draw) & (w > 0))
        some = torch.nonzero(w > 0)
        out.append(toks[:n] + [int(hit[0]) if len(hit) else int(some[-1]) if len(some) else -1] + [-1] * (K - n))
        count.append(n)
        near.append(float((c - draw).abs().min() / c[-1]) if float(c[-1]) > 0 and math.isfinite(draw) else 1.0)
    return torch.tensor(out, device=DEV), torch.tensor(count, device=DEV), min(near) if near else 1.0


def _case(B, K, V, dtype, draft=True, seed=0, sharp=2.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    z = torch.randn(B, K + 1, V, generator=g, device=DEV) * sharp
    q = torch.softmax(z[:, :K], -1).to(dtype)
    p = torch.softmax(z + 0.7 * torch.randn(z.shape, generator=g, device=DEV), -1).to(dtype)
    x = torch.multinomial(q.reshape(B * K, V).float().clamp_min(1e-30), 1, generator=g).view(B, K) if B * K else \
        torch.zeros(B, K, dtype=torch.long, device=DEV)
    return p, q if draft else None, x, torch.rand(B, K + 1, generator=g, device=DEV)


def _check(p, q, x, u):
    """Equal, tokens and counts.  A drawn number within 1e-12 of a border could go to either side (sums of V 64-bit terms
    differ by up to V 2^-53 of their value between orders); none does here."""
    from epure import sampling
    got, n = sampling.verify(p, q, x, u)
    want, count, near = _expected(p, q, x, u)
    assert near > 1e-12 or float(u.max()) in (0.0, 1.0)
    assert torch.equal(n, count) and torch.equal(got, want)
    again = sampling.verify(p, q, x, u)
    assert torch.equal(again[0], got) and torch.equal(again[1], n)
    return got, n


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("draft", [True, False])
@pytest.mark.parametrize("B,K,V", [(1, 4, 151936), (3, 1, 1), (5, 2, 2), (4, 3, 33), (7, 5, 1000), (2, 0, 4097), (9, 40, 130),
                                   (33, 7, 32001), (200, 2, 511), (1, 8, 300000), (16, 4, 128)])
def test_verify(dtype, draft, B, K, V):
    _check(*_case(B, K, V, dtype, draft))


def test_every_outcome_occurs():
    """Accepted rows, rows refused at each place, by the thousand."""
    _, n = _check(*_case(2000, 3, 50, torch.float32, sharp=1.0))
    assert set(n.tolist()) == {0, 1, 2, 3}


def test_ragged_drafts():
    """A row's drafts end at its first negative token; nothing is refused there."""
    p, q, x, u = _case(12, 5, 700, torch.float32, seed=2)
    for b in range(12):
        x[b, b % 6:] = torch.where(torch.arange(5 - b % 6, device=DEV) % 2 == 0, -1, x[b, b % 6:]) if b % 6 < 5 else x[b, 5:]
    for d in (q, None):
        got, n = _check(p, d, x, u)
        assert bool((n <= torch.arange(12, device=DEV) % 6).all())


@pytest.mark.parametrize("V", [1000, 32001, 40000])
def test_borders(V):
    """u of 0 takes the first token with a weight, 1 the last; a draft with u q = p is refused, u of 0 accepts whatever the
    target gives a weight."""
    p, q, x, u = _case(6, 2, V, torch.float32, seed=3)
    p[:, :, :5] = 0
    p[:, :, -3:] = 0
    q[:, :, -3:] = 0
    u[0] = 0
    u[1] = 1
    u[2, 2], u[3, 2] = 0, 1
    _check(p, q, x, u)
    _check(p, None, x, u)
    p[:, :2], u[:, :2] = q, 1.0                        # u q = p: refused, and no residual: p itself
    got, n = _check(p, q, x, u)
    assert not n.any()
    x[:] = 2                                           # a draft that neither model gives a weight
    p[:, :, 2] = 0
    q[:, :, 2] = 0
    got, n = _check(p, q, x, u)
    assert not n.any()


def test_weights_that_are_not_ordinary():
    """Negative weights and NaN count as nothing, rows that sum to another number than 1 keep their proportions, a row
    without any weight gives -1."""
    p, q, x, u = _case(8, 2, 3000, torch.float32, seed=4)
    p[0, :, ::7] = math.nan
    q[1, :, ::5] = math.nan
    p[2, :, ::3] *= -1
    p[3] *= 1e-30
    p[4] *= 1e30
    p[5] = 0
    p[6, 0, 17] = math.inf
    x[0, 0] = 7                                        # a NaN probability is not above anything
    u[6] = 0.5
    got, n = _check(p, q, x, u)
    assert got[5].tolist() == [-1, -1, -1]
    _check(p, None, x, u)
    tiny = torch.full((1, 1, 100000), 2.0 ** -140, device=DEV)      # subnormal weights
    _check(tiny, None, torch.zeros(1, 0, dtype=torch.long, device=DEV), torch.tensor([[0.7]], device=DEV))


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("V", [1, 4, 999, 32001, 150000])
def test_nothing_left_but_the_draft(dtype, V):
    """Drafts without probabilities whose target gives a weight to nothing else: a refused one leaves nothing, so the target
    itself is drawn from, which is the drafted token.  (Filtered probabilities that were not normalised again, or a
    float16 row whose others went to 0.)"""
    g = torch.Generator(device=DEV).manual_seed(11)
    x = torch.randint(0, V, (8, 3), generator=g, device=DEV)
    x[0], x[1] = 0, V - 1
    p = torch.zeros(8, 4, V, dtype=dtype, device=DEV)
    p[:, :3].scatter_(2, x[:, :, None], 0.5)
    p[:, 3, V // 2] = 0.25
    p[4] *= -1                                         # no weight at all
    p[5, 0] = torch.where(p[5, 0] == 0, math.nan, p[5, 0].float()).to(dtype)
    u = torch.full((8, 4), 0.7, device=DEV)
    u[2, 0], u[3, :2] = 0.3, 0.3                       # refused at the second and the third draft
    u[:, 3] = torch.tensor([0.3, 0.999, 0.3, 0.001, 0.3, 0.3, 0.6, 0.9], device=DEV)
    got, n = _check(p, None, x, u)
    assert n.tolist() == [0, 0, 1, 2, 0, 0, 0, 0]
    for b in (0, 1, 2, 3, 5, 6, 7):
        assert int(got[b, n[b]]) == int(x[b, n[b]])
    assert got[4].tolist() == [-1] * 4


def test_close_weights_need_64_bits():
    """A uniform row of 2^18 tokens: every number's token is where it says, not where float32 sums would put it."""
    from epure import sampling
    V = 1 << 18
    p = torch.full((512, 1, V), 2.0 ** -18, device=DEV)
    at = torch.randint(0, V, (512, 1), generator=torch.Generator(device=DEV).manual_seed(5), device=DEV)
    u = (at.double() / V).float()                      # exact: the cumulative sum passes it at token `at`
    got, _ = sampling.verify(p, None, torch.zeros(512, 0, dtype=torch.long, device=DEV), u)
    assert torch.equal(got, at)


def test_layouts():
    """Strided rows and steps, a broadcast target, probabilities that no wide load can take, tokens of a wider table."""
    from epure import sampling
    for dtype in (torch.float32, torch.bfloat16):
        p, q, x, u = _case(6, 3, 999, dtype, seed=6)
        want = _check(p, q, x, u)
        for shift in (1, 3, 4, 8):
            wide = torch.zeros(6, 7, 999 + 24, dtype=dtype, device=DEV)
            wide[:, 2:6, shift:shift + 999] = p
            far = torch.zeros(6 * 3 * 999 + 5, dtype=dtype, device=DEV)[5:].view(6, 3, 999).copy_(q)
            got = sampling.verify(wide[:, 2:6, shift:shift + 999], far, x, u)
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        other = torch.empty(4, 6, 999, dtype=dtype, device=DEV).transpose(0, 1).copy_(p)
        table = torch.full((6, 9), -7, device=DEV)
        table[:, 4:7] = x
        many = torch.zeros(6, 8, device=DEV)
        many[:, :4] = u
        got = sampling.verify(other, q, table[:, 4:7], many[:, :4])
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        _check(p[:1].expand(6, 4, 999), None, x, u)
    none = sampling.verify(p[:0], q[:0], x[:0], u[:0])
    assert none[0].shape == (0, 4) and none[1].shape == (0,)


def test_distribution():
    """Over many rows the first token is distributed as the target, whatever the draft: within 5 standard deviations of
    each token's count."""
    from epure import sampling
    g = torch.Generator(device=DEV).manual_seed(7)
    N, V = 200000, 8
    p = torch.softmax(torch.randn(1, 2, V, generator=g, device=DEV), -1).expand(N, 2, V)
    q = torch.softmax(torch.randn(1, 1, V, generator=g, device=DEV), -1).expand(N, 1, V)
    x = torch.multinomial(q[0, 0], N, replacement=True, generator=g)[:, None]
    tokens, _ = sampling.verify(p, q, x, torch.rand(N, 2, generator=g, device=DEV))
    seen = torch.bincount(tokens[:, 0], minlength=V).double()
    expect = p[0, 0].double() * N
    assert bool(((seen - expect).abs() <= 5 * (expect * (1 - p[0, 0].double())).sqrt()).all())


def test_captured():
    from epure import sampling
    p, q, x, u = _case(4, 3, 5000, torch.float32, seed=8)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        sampling.verify(p, q, x, u)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = sampling.verify(p, q, x, u)
    for seed in (9, 10):
        for t, new in zip((p, q, x, u), _case(4, 3, 5000, torch.float32, seed=seed)):
            t.copy_(new)
        graph.replay()
        want = _expected(p, q, x, u)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_refusals():
    from epure import sampling
    p, q, x, u = _case(2, 3, 100, torch.float32)
    for bad in (dict(q=q.half()), dict(q=q[:, :2]), dict(q=q[..., :99]), dict(x=x.int()), dict(x=x[:, :2]), dict(u=u[:, :3]),
                dict(u=u.double()), dict(p=p[:, :, ::2]), dict(p=p[0]), dict(x=x.cpu()), dict(q=q.cpu()), dict(u=u.cpu())):
        with pytest.raises(RuntimeError, match="must be"):
            sampling.verify(*{**dict(p=p, q=q, x=x, u=u), **bad}.values())
    with pytest.raises(TypeError, match="dtype"):
        sampling.verify(p.double(), None, x, u)
    with pytest.raises(TypeError, match="tensor"):
        sampling.verify(p, q, x.tolist(), u)
    with pytest.raises(RuntimeError, match="CUDA"):
        sampling.verify(p.cpu(), None, x, u)


_CHILD = r"""
import sys, torch
sys.path.insert(0, sys.argv[1])
from epure import _native, sampling
p = torch.full((2, 3, 10), 0.1, device="cuda:0")
x = torch.tensor([[4, 10], [10, 3]], device="cuda:0")
u = torch.tensor([[0.0, 0.0, 0.35]] * 2, device="cuda:0")
got, n = sampling.verify(p, None, x, u)
assert got.tolist() == [[4, 3, -1], [3, -1, -1]] and n.tolist() == [1, 0]
torch.cuda.synchronize()
print("FLAG", _native.device_error())
"""


def test_tokens_outside_the_vocabulary_are_reported():
    """They end their row's drafts (in a child process: the flag stays set)."""
    r = subprocess.run([sys.executable, "-c", _CHILD, PKG], capture_output=True, text=True, timeout=300, env=dict(os.environ))
    assert r.returncode == 0, r.stderr[-2000:]
    assert "FLAG 8" in r.stdout


_BEHIND = r"""
import sys, torch
sys.path.insert(0, sys.argv[1])
from epure import _native, sampling
p = torch.full((3, 41, 10), 0.1, device="cuda:0")
u = torch.full((3, 41), 0.35, device="cuda:0")
x = torch.full((3, 40), 4, device="cuda:0")
x[0, 2], x[0, 3] = -1, 10                              # behind a row's end
x[1, 39], x[1, 7:39] = 2 ** 40, -1
x[2, 0] = -5
x[2, 1:] = 77
u[0, :2] = 0.0
got, n = sampling.verify(p, None, x, u)
assert n.tolist() == [2, 0, 0]
assert _native.device_error() == 0
x[1] = 4                                               # refused at once, far before the one outside
x[1, 38] = 10
sampling.verify(p, None, x, u)
torch.cuda.synchronize()
print("FLAG", _native.device_error())
"""


def test_what_lies_behind_a_rows_drafts_is_not_reported():
    """Tokens behind a row's end are no drafts, whatever they hold; one of the row's drafts that is outside the vocabulary is
    reported wherever it lies and whatever was refused before it."""
    r = subprocess.run([sys.executable, "-c", _BEHIND, PKG], capture_output=True, text=True, timeout=300, env=dict(os.environ))
    assert r.returncode == 0, r.stderr[-2000:]
    assert "FLAG 8" in r.stdout
