"""The paged and rotary calls beside autograd: nothing is detached or overwritten without a word."""
import pytest
import torch
import torch.autograd.forward_ad as fwd
from test_gpu_paged import DEV, _fill, _gpu, _pages, _tokens  # noqa: F401 (_gpu: a fixture)

pytestmark = pytest.mark.gpu


def _rows(*heads, grad=False):
    return [torch.randn(4, h, 64, device=DEV).to(torch.bfloat16).requires_grad_(grad) for h in heads]


def _cache():
    pages = _pages([4], 2, 64, 16, "same", torch.bfloat16)
    return (pages, *_tokens([4]))


def test_gradients_that_would_be_lost_are_refused():
    from epure import paged, rotary
    pages, seq, pos = _cache()
    cos, sin = rotary.rope_tables(64, 8, DEV)
    (q, k, v), (gq, gk, gv) = _rows(4, 2, 2), _rows(4, 2, 2, grad=True)
    _fill(pages, [4], torch.bfloat16)
    n = torch.tensor([4], device=DEV)
    page = int(pages.table[0, 0])
    before = [pages.k[page, :, :4].clone(), pages.v[page, :, :4].clone()]
    for call in (lambda: rotary.rope(gq, None, pos, cos, sin, out=torch.empty_like(q)),
                 lambda: rotary.rope(q, k, pos, cos, sin, out=(q, gk * 1)),
                 lambda: rotary.rope(q, None, pos, cos.clone().requires_grad_(True), sin),
                 lambda: rotary.rope(gq, None, pos, cos, sin.clone().requires_grad_(True)),
                 lambda: paged.write(pages, gk, v, seq, pos), lambda: paged.write(pages, k, gv, seq, pos),
                 lambda: paged.write(pages, k, v, seq, pos, q=gq),
                 lambda: paged.write(pages, k, v, seq, pos, q=q, q_out=gq * 1),
                 lambda: paged.attend(pages, gq[:1], n),
                 lambda: paged.attend(pages, q[:1], n, out=(gq * 1)[:1])):
        with pytest.raises(RuntimeError, match="gradient"):
            call()
    assert torch.equal(pages.k[page, :, :4], before[0]) and torch.equal(pages.v[page, :, :4], before[1])


def test_without_grad_mode_they_are_taken():
    from epure import paged, rotary
    pages, seq, pos = _cache()
    cos, sin = rotary.rope_tables(64, 8, DEV)
    gq, gk, gv = _rows(4, 2, 2, grad=True)
    q, k, v = (t.detach().clone() for t in (gq, gk, gv))
    n = torch.tensor([4], device=DEV)
    want = paged.write(pages, k, v, seq, pos, q=q, cos=cos, sin=sin)
    att = paged.attend(pages, want[:1], n)
    with torch.no_grad():
        assert torch.equal(paged.write(pages, gk, gv, seq, pos, q=gq, cos=cos, sin=sin), want)
        assert torch.equal(rotary.rope(gq, None, pos, cos, sin, out=torch.empty_like(q)), want)
        assert torch.equal(paged.attend(pages, gq[:1], n), paged.attend(pages, q[:1], n))
    with torch.inference_mode():
        assert torch.equal(paged.attend(pages, want[:1], n), att)
    x = gq.detach().requires_grad_(True)               # the gradient itself is as before
    (dx,) = torch.autograd.grad(rotary.rope(x, None, pos, cos, sin), x, q)
    assert torch.equal(dx, rotary.rope(q, None, pos, cos, sin, inverse=True))


def test_forward_mode_tangents_are_refused():
    from epure import paged, rotary
    pages, seq, pos = _cache()
    cos, sin = rotary.rope_tables(64, 8, DEV)
    q, k, v = _rows(4, 2, 2)
    _fill(pages, [4], torch.bfloat16)
    with fwd.dual_level():
        dual = fwd.make_dual(q, torch.ones_like(q))
        for call in (lambda: rotary.rope(dual, None, pos, cos, sin),
                     lambda: rotary.rope(dual, k, pos, cos, sin, out=(torch.empty_like(q), torch.empty_like(k))),
                     lambda: paged.write(pages, k, v, seq, pos, q=dual),
                     lambda: paged.attend(pages, dual[:1], torch.tensor([4], device=DEV))):
            with pytest.raises(RuntimeError, match="tangent"):
                call()
        assert torch.isfinite(rotary.rope(q, None, pos, cos, sin).float()).all()


def test_writes_are_counted():
    """A tensor that an earlier operation saved for its backward, overwritten in place: torch's own error."""
    from epure import paged, rotary
    pages, seq, pos = _cache()
    cos, sin = rotary.rope_tables(64, 8, DEV)
    q, k, v = _rows(4, 2, 2)
    n = torch.tensor([4], device=DEV)

    def versions():
        return [t._version for t in (q, k, pages.k, pages.v)]

    before = versions()
    rotary.rope(q, k, pos, cos, sin)
    paged.read(pages, seq, pos)
    assert versions() == before
    rotary.rope(q, k, pos, cos, sin, out=(q, k))
    assert versions() == [before[0] + 1, before[1] + 1, before[2], before[3]]
    paged.write(pages, k, v, seq, pos, q=q, q_out=q)
    assert versions() == [before[0] + 2, before[1] + 1, before[2] + 1, before[3] + 1]
    out = torch.empty_like(q[:1])
    paged.attend(pages, q[:1], n, out=out)
    assert out._version == 1 and versions()[0] == before[0] + 2
    q8 = _pages([4], 2, 64, 16, "int8", torch.bfloat16)
    scale = q8.k_scale._version
    paged.write(q8, k, v, seq, pos)
    assert q8.k_scale._version == scale + 1
    w = torch.randn(64, 64, device=DEV, dtype=torch.bfloat16, requires_grad=True)
    for overwrite in (lambda t: rotary.rope(t, None, pos, cos, sin, out=t),
                      lambda t: paged.write(pages, k, v, seq, pos, q=t, q_out=t)):
        x = torch.randn(4, 4, 64, device=DEV, dtype=torch.bfloat16)
        y = x @ w                                      # saves x
        overwrite(x)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.sum().backward()


def test_inference_tensors_are_taken():
    from epure import paged
    with torch.inference_mode():
        pages, seq, pos = _cache()
        _, k, v = _rows(4, 2, 2)
    paged.write(pages, k, v, seq, pos)
    got = paged.read(pages, seq, pos)
    assert torch.equal(got[0], k) and torch.equal(got[1], v)
