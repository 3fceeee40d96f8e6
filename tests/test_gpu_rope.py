"""Rotary positions (epq_rope) against the rotation in 64 bits, its gradient against differences, its refusals."""
import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
# Unit roundoff of each type: results are rounded once from float32.
ROUND = {torch.float32: 0.0, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from epure import _native
    _native.load_library()
    yield
    assert _native.device_error() == 0


def _exact(x, pos, cos, sin, interleaved):
    x, r = x.double(), 2 * cos.shape[1]
    c, s = cos.double()[pos][:, None], sin.double()[pos][:, None]
    a, b = (slice(0, r, 2), slice(1, r, 2)) if interleaved else (slice(0, r // 2), slice(r // 2, r))
    y = x.clone()
    y[..., a] = x[..., a] * c - x[..., b] * s
    y[..., b] = x[..., b] * c + x[..., a] * s
    return y


def _inputs(m, heads, kv, hd, r, dtype, seed=0, max_len=997, fused=True):
    from epure.rotary import rope_tables
    g = torch.Generator(device=DEV).manual_seed(seed)
    cos, sin = rope_tables(r, max_len, DEV, theta=5e5, scaling="yarn", factor=4.0)
    pos = torch.randint(0, max_len, (m,), generator=g, device=DEV)
    qkv = torch.randn(m, heads + 2 * kv, hd, generator=g, device=DEV).to(dtype)
    q, k = qkv[:, :heads], qkv[:, heads:heads + kv]
    return (q, k) if fused else (q.contiguous(), k.contiguous()), pos, cos, sin


def _close(got, want):
    # one rounding to the type, and three float32 roundings (two products, their sum) of
    # values of at most |a c| + |b s| <= sqrt(2) gain |(a, b)| < 3 max|x|
    slack = 3 * 2.0 ** -24 * 3 * float(want.abs().max())
    err = (got.double() - want).abs()
    assert bool((err <= ROUND[got.dtype] * want.abs() + slack + 2.0 ** -25).all()), float(err.max())


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("heads,kv,hd,r", [(32, 8, 128, 128), (8, 2, 64, 64), (12, 4, 80, 32), (4, 4, 128, 6),
                                           (3, 1, 96, 50), (2, 1, 256, 256), (1, 1, 2, 2), (5, 0, 33, 32),
                                           (2, 2, 1000, 16), (6, 3, 10, 10)])
@pytest.mark.parametrize("m", [1, 37])
def test_rope_matches_definition(dtype, interleaved, heads, kv, hd, r, m):
    from epure import rotary
    (q, k), pos, cos, sin = _inputs(m, heads, kv, hd, r, dtype)
    if kv == 0:
        k = None
    got = rotary.rope(q, k, pos, cos, sin, interleaved=interleaved)
    back = rotary.rope(q, k, pos, cos, sin, interleaved=interleaved, inverse=True)
    for x, y, z in ((q, got[0], back[0]), (k, got[1], back[1])) if k is not None else ((q, got, back),):
        assert y.shape == x.shape and y.dtype == dtype
        _close(y, _exact(x, pos, cos, sin, interleaved))
        _close(z, _exact(x, pos, cos, -sin, interleaved))
        assert torch.equal(y[..., r:], x[..., r:])


@pytest.mark.parametrize("m", [3000, 20000])
def test_many_rows_match_tensor_formula_bit_for_bit(m):
    """The half layout equals x1 c - x2 s, x2 c + x1 s written with float32 tensors."""
    from epure import rotary
    (q, k), pos, cos, sin = _inputs(m, 16, 8, 128, 128, torch.bfloat16)
    got = rotary.rope(q, k, pos, cos, sin)
    c, s = cos[pos][:, None], sin[pos][:, None]
    for x, y in zip((q, k), got):
        f = x.float()
        a, b = f[..., :64], f[..., 64:]
        assert torch.equal(y, torch.cat([a * c - b * s, b * c + a * s], -1).to(x.dtype))


def test_in_place_empty_and_unaligned():
    from epure import rotary
    (q, k), pos, cos, sin = _inputs(19, 8, 2, 64, 64, torch.bfloat16, fused=False)
    want = rotary.rope(q, k, pos, cos, sin)
    q2, k2 = q.clone(), k.clone()
    got = rotary.rope(q2, k2, pos, cos, sin, out=(q2, k2))
    assert got[0] is q2 and torch.equal(q2, want[0]) and torch.equal(k2, want[1])
    none = rotary.rope(q[:0], k[:0], pos[:0], cos, sin)
    assert none[0].shape == (0, 8, 64)
    flat = torch.zeros(q.numel() + 1, dtype=q.dtype, device=DEV)
    odd = flat[1:].view(q.shape)                       # 2-byte aligned
    odd.copy_(q)
    assert torch.equal(rotary.rope(odd, None, pos, cos, sin), want[0])
    wide = torch.zeros(19, 8, 70, dtype=q.dtype, device=DEV)[..., 3:67]     # odd head stride
    wide.copy_(q)
    assert torch.equal(rotary.rope(wide, None, pos, cos, sin), want[0])


@pytest.mark.parametrize("interleaved", [False, True])
def test_gradient(interleaved):
    """Against the formula's gradient, and against central differences of the call itself: the rotation is
    linear, so a difference over a step h is exact but for float32 rounding of its two results,
    2 * 2^-24 * |y| * 3 / (2 h)."""
    from epure import rotary
    (q, k), pos, cos, sin = _inputs(5, 3, 2, 16, 8, torch.float32)
    q, k = q.clone().requires_grad_(True), k.clone().requires_grad_(True)
    g = torch.Generator(device=DEV).manual_seed(3)
    dyq, dyk = torch.randn(q.shape, generator=g, device=DEV), torch.randn(k.shape, generator=g, device=DEV)
    yq, yk = rotary.rope(q, k, pos, cos, sin, interleaved=interleaved)
    dq, dk = torch.autograd.grad((yq, yk), (q, k), (dyq, dyk))
    _close(dq, _exact(dyq, pos, cos, -sin, interleaved))
    _close(dk, _exact(dyk, pos, cos, -sin, interleaved))
    h = 0.5
    with torch.no_grad():
        for i in (0, 3, 7, 9, 15):
            e = torch.zeros_like(q)
            e[:, 1, i] = h
            up, _ = rotary.rope(q + e, k, pos, cos, sin, interleaved=interleaved)
            down, _ = rotary.rope(q - e, k, pos, cos, sin, interleaved=interleaved)
            slope = ((up.double() - down.double()) / (2 * h) * dyq.double()).sum((1, 2))
            bound = 16 * 4 * 2.0 ** -24 * 6 * float(up.abs().max()) * float(dyq.abs().max()) / (2 * h)
            assert float((slope - dq[:, 1, i].double()).abs().max()) <= bound


def test_gradient_of_one_used_output():
    """Only q's output is used: k's gradient is zero."""
    from epure import rotary
    (q, k), pos, cos, sin = _inputs(5, 3, 2, 16, 16, torch.float32)
    q, k = q.clone().requires_grad_(True), k.clone().requires_grad_(True)
    yq, _ = rotary.rope(q, k, pos, cos, sin)
    yq.sum().backward()
    _close(q.grad, _exact(torch.ones_like(q), pos, cos, -sin, False))
    assert not k.grad.any()


@pytest.mark.parametrize("with_k", [True, False])
def test_gradient_of_a_gradient(with_k):
    """d/dq of w . (R^T R q) is R^T R w: two rotations, each with three float32 roundings of values below
    3 max|w| (the gain of these tables is under 1.2), the first's error turned by the second."""
    from epure import rotary
    (q, k), pos, cos, sin = _inputs(5, 3, 2, 16, 8, torch.float32)
    q = q.clone().requires_grad_(True)
    y = rotary.rope(q, k if with_k else None, pos, cos, sin)
    y = y[0] if with_k else y
    (dq,) = torch.autograd.grad((y * y).sum() / 2, q, create_graph=True)        # R^T R q
    w = torch.randn(q.shape, generator=torch.Generator(device=DEV).manual_seed(4), device=DEV)
    (d2,) = torch.autograd.grad((dq * w).sum(), q)                              # R^T R w
    want = _exact(_exact(w, pos, cos, sin, False), pos, cos, -sin, False)
    assert float((d2.double() - want).abs().max()) <= 3 * 2.0 ** -24 * 3 * float(w.abs().max()) * (1 + 2)


def test_graph_replays_at_new_positions():
    from epure import rotary
    (q, k), pos, cos, sin = _inputs(16, 8, 2, 64, 64, torch.bfloat16, fused=False)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        rotary.rope(q, k, pos, cos, sin)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = rotary.rope(q, k, pos, cos, sin)
    pos.copy_((pos + 11) % 997)
    graph.replay()
    _close(out[0], _exact(q, pos, cos, sin, False))
    _close(out[1], _exact(k, pos, cos, sin, False))


def test_refusals():
    from epure import rotary
    (q, k), pos, cos, sin = _inputs(4, 4, 2, 32, 32, torch.bfloat16, fused=False)
    with pytest.raises(RuntimeError, match="CUDA"):
        rotary.rope(q.cpu(), None, pos, cos, sin)
    with pytest.raises(TypeError, match="not supported"):
        rotary.rope(q.double(), None, pos, cos, sin)
    with pytest.raises(RuntimeError, match="pos"):
        rotary.rope(q, k, pos.int(), cos, sin)
    with pytest.raises(RuntimeError, match="pos"):
        rotary.rope(q, k, pos[:3], cos, sin)
    with pytest.raises(RuntimeError, match="tables"):
        rotary.rope(q, k, pos, cos.double(), sin.double())
    with pytest.raises(RuntimeError, match="rotary tables"):
        rotary.rope(q[..., :16].contiguous(), None, pos, cos, sin)
    with pytest.raises(RuntimeError, match="rope input"):
        rotary.rope(q, k.float(), pos, cos, sin)
    with pytest.raises(RuntimeError, match="contiguous"):
        rotary.rope(q.transpose(1, 2).contiguous().transpose(1, 2), None, pos, cos, sin)


_CHILD = r"""
import sys, torch
sys.path.insert(0, sys.argv[1])
from epure import _native, rotary
q = torch.randn(4, 2, 32, device="cuda:0")
cos, sin = rotary.rope_tables(32, 10, "cuda:0")
assert _native.device_error() == 0
y = rotary.rope(q, None, torch.tensor([0, 10, -1, 9], device="cuda:0"), cos, sin)
torch.cuda.synchronize()
assert not y[1].any() and not y[2].any() and y[0].any() and y[3].any()
print("FLAG", _native.device_error())
"""


def test_position_past_the_table_is_reported():
    """Zeros and bit 4 of epq_device_error (in a child process: the flag stays set)."""
    import subprocess
    import sys
    from conftest import PKG
    r = subprocess.run([sys.executable, "-c", _CHILD, PKG], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "FLAG 16" in r.stdout, r.stdout + r.stderr[-2000:]
