"""Layouts of the paged and rotary calls' tensors (outputs in other orders, strides that say nothing), and flags that
have no truth value."""
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


@pytest.mark.parametrize("fmt", ["same", "int8"])
def test_strides_of_single_elements_say_nothing(fmt):
    """One page, one key head, slot, table column, row or head, with strides that no dense tensor has."""
    from epure import paged
    g = torch.Generator(device=DEV).manual_seed(52)

    def odd(t, dim, stride=7):
        assert t.shape[dim] == 1
        return t.as_strided(t.shape, [stride if d == dim else s for d, s in enumerate(t.stride())])

    for pages, kv, ps, seqs in ((1, 2, 16, 1), (3, 1, 16, 3), (3, 2, 1, 3)):
        plain = _pages([min(ps, 5)] * seqs, kv, 64, ps, fmt, torch.bfloat16, spare=pages - seqs)
        dim = 0 if pages == 1 else 1 if kv == 1 else 2
        strange = [t if t is None else odd(t, dim) for t in (plain.k, plain.v, plain.k_scale, plain.v_scale)]
        table = odd(plain.table, 1 if seqs > 1 else 0)
        assert table.shape == plain.table.shape and table.stride() != plain.table.stride()
        cache = paged.KVPages(strange[0], strange[1], table, *strange[2:])
        m = seqs
        seq, pos = torch.arange(m, dtype=torch.int32, device=DEV), torch.zeros(m, dtype=torch.long, device=DEV)
        x = torch.randn(m, 2, kv, 64, generator=g, device=DEV).to(torch.bfloat16)
        q = torch.randn(m, 2 * kv, 64, generator=g, device=DEV).to(torch.bfloat16)
        rows = (x[:, 0], x[:, 1]) if m > 1 else (odd(x[:, 0], 0), odd(x[:, 1], 0))
        got = [paged.write(c, *rows, seq, pos, q=q if m > 1 else odd(q, 0)) for c in (plain, cache)]
        assert torch.equal(got[0], got[1]) and torch.equal(got[0], q)
        n = torch.ones(m, dtype=torch.long, device=DEV)
        for a, b in zip(paged.read(plain, seq, pos), paged.read(cache, seq, pos)):
            assert torch.equal(a, b)
        assert torch.equal(paged.attend(plain, q, n), paged.attend(cache, q if m > 1 else odd(q, 0), n))


def test_real_strides_are_still_refused():
    from epure import paged
    pages, seq, pos, q, k, v, cos, sin = _inputs()
    two = _pages([20, 20], 2, 64, 16, "int8", torch.bfloat16)
    for bad in (pages._replace(v=pages.v[:, :, ::2]), pages._replace(k=pages.k.transpose(1, 2), v=pages.v.transpose(1, 2)),
                pages._replace(v=torch.empty(3, 2, 2, 16, 64, dtype=q.dtype, device=DEV)[:, 0]),
                two._replace(table=two.table.t().contiguous().t()),
                two._replace(v_scale=torch.empty(*two.v_scale.shape[:2], 32, device=DEV)[..., ::2])):
        assert bad.k.shape[0] > 1
        with pytest.raises(RuntimeError, match="alike|contiguous|page table"):
            paged.read(bad, seq, pos)


def test_flags_without_a_truth_value():
    """The flag's own exception, and nothing is written."""
    from epure import paged, rotary
    pages, seq, pos, q, k, v, cos, sin = _inputs()
    paged.write(pages, k, v, seq, pos)
    before = pages.k.clone().nan_to_num_(9.0)
    out = torch.zeros_like(q)
    both = torch.tensor([True, False])
    for call in (lambda: rotary.rope(q, None, pos, cos, sin, interleaved=both, out=out),
                 lambda: rotary.rope(q, None, pos, cos, sin, inverse=both, out=out),
                 lambda: paged.write(pages, v, k, seq, pos, cos=cos, sin=sin, interleaved=both),
                 lambda: paged.write(pages, v, k, seq, pos, qk_norm=both),
                 lambda: paged.attend(pages, q[:1], pos[1:2], return_lse=both)):
        with pytest.raises(RuntimeError, match="ambiguous"):
            call()
    assert not out.any() and torch.equal(pages.k.nan_to_num(9.0), before)
    assert torch.equal(rotary.rope(q, None, pos, cos, sin, interleaved=torch.tensor(True)),
                       rotary.rope(q, None, pos, cos, sin, interleaved=True))


def test_an_output_without_its_input_is_refused():
    from epure import paged
    pages, seq, pos, q, k, v, cos, sin = _inputs()
    with pytest.raises(RuntimeError, match="q_out needs q"):
        paged.write(pages, k, v, seq, pos, q_out=torch.empty_like(q))
