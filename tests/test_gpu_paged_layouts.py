"""Layouts of the paged and rotary calls' tensors: outputs in other orders, strides that say nothing."""
import pytest
import torch
from test_gpu_paged import DEV, _gpu, _pages, _tokens  # noqa: F401 (_gpu: a fixture)

pytestmark = pytest.mark.gpu


def _inputs():
    from epure import rotary
    pages = _pages([6], 2, 64, 16, "same", torch.bfloat16)
    x = torch.randn(6, 8, 64, generator=torch.Generator(device=DEV).manual_seed(51), device=DEV).to(torch.bfloat16)
    return (pages, *_tokens([6]), x[:, :4], x[:, 4:6], x[:, 6:], *rotary.rope_tables(64, 8, DEV))


def test_outputs_of_heads_by_rows_and_of_interleaved_rows():
    from epure import paged, rotary
    pages, seq, pos, q, k, v, cos, sin = _inputs()
    want = rotary.rope(q, None, pos, cos, sin)
    for out in (torch.empty(4, 6, 64, dtype=q.dtype, device=DEV).transpose(0, 1),
                torch.empty(6, 5, 80, dtype=q.dtype, device=DEV)[:, :4, :64],
                torch.empty(6, 2, 4, 64, dtype=q.dtype, device=DEV)[:, 0],
                torch.empty(4, 64, 6 * 64, dtype=q.dtype, device=DEV)[:, 0].view(4, 6, 64).transpose(0, 1)):
        rotary.rope(q, None, pos, cos, sin, out=out.zero_())
        assert torch.equal(out, want)
        assert torch.equal(paged.write(pages, k, v, seq, pos, q=q, q_out=out.zero_(), cos=cos, sin=sin), want)
    whole = q.clone()
    first = whole[:1]                                  # one row: its stride says nothing
    rotary.rope(first, None, pos[:1], cos, sin, out=first)
    assert torch.equal(whole[:1], want[:1]) and torch.equal(whole[1:], q[1:])


def test_outputs_whose_rows_are_one_are_refused():
    from epure import paged, rotary
    pages, seq, pos, q, k, v, cos, sin = _inputs()
    one = torch.zeros(1, 4, 64, dtype=q.dtype, device=DEV)
    head = torch.zeros(6, 1, 64, dtype=q.dtype, device=DEV)
    for out in (one.expand(6, 4, 64), head.expand(6, 4, 64)):
        with pytest.raises(RuntimeError, match="overlap"):
            rotary.rope(q, None, pos, cos, sin, out=out)
        with pytest.raises(RuntimeError, match="overlap"):
            paged.write(pages, k, v, seq, pos, q=q, q_out=out)
    flat = q.contiguous().view(-1)
    with pytest.raises(RuntimeError, match="overlap"):
        rotary.rope(flat.view(6, 4, 64), None, pos, cos, sin, out=flat.view(4, 6, 64).transpose(0, 1))
    assert not one.any() and not head.any()
    # inputs may be expanded
    same = rotary.rope(q[:1].expand(6, 4, 64), None, pos, cos, sin)
    assert torch.equal(same, rotary.rope(q[:1].expand(6, 4, 64).contiguous(), None, pos, cos, sin))
