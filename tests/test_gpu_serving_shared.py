"""The decoder's steps on the shared form of attention itself: calls that share whatever can be, each shown to have read the
prefix through the first row's pages alone, and a batch large enough to share by the reckoning."""
import functools

import pytest
import torch
from test_gpu_serving import DEV, _decoder, _gpu, _prompts  # noqa: F401 (_gpu: a fixture)
from test_gpu_serving_drafts import _close, _wide

pytestmark = pytest.mark.gpu


@pytest.fixture
def always(monkeypatch):
    """attend_shared shares whatever can be; counts its calls."""
    from epure import paged
    real, calls = paged.attend_shared, []

    @functools.wraps(real)
    def call(*a, **kw):
        calls.append(1)
        return real(*a, **{**kw, "always": True})

    monkeypatch.setattr(paged, "attend_shared", call)
    return calls


def _one_set_of_pages(b, rows, tokens):
    """Lets the tables of all sequences but the first name a page of zeros for the first `tokens` tokens: only what is read
    through the first one's is right then."""
    zero = b.cache._free[-1]
    for pages in b._layers:
        for x in (pages.k, pages.v, pages.k_scale, pages.v_scale):
            if x is not None:
                x[zero].zero_()
    b.cache.table[1:rows, :tokens // b.cache.page_size] = zero


def _behind_a_prefix(b, rows, prefix, own):
    """Sequences behind one prefix of whole pages, row i with own[i] tokens more and room for 8."""
    n = len(prefix)
    b.cache.reserve(0, n + own[0] + 8)
    b.prefill(0, prefix)
    for i in range(1, rows):
        assert b.cache.share(i, 0, n) == n
        b.cache.reserve(i, n + own[i] + 8)
    for i in range(rows):
        b.prefill(i, (torch.arange(own[i]) * 91 + i) % 1000, past=n)


@pytest.mark.parametrize("fmt", ["same", "int8", "fp8"])
def test_step_reads_the_prefix_once(fmt, always):
    from epure.serving import BatchDecoder
    b = BatchDecoder(_decoder(), seqs=7, format=fmt, page_size=16)
    _behind_a_prefix(b, 6, _prompts([64])[0], [3, 1, 9, 16, 2, 5])
    seq = torch.arange(6, dtype=torch.int32, device=DEV)
    tok = torch.arange(6, device=DEV) * 130
    pos = torch.tensor([67, 65, -1, 80, 66, 69], device=DEV)
    shared = (torch.tensor([0, 6], dtype=torch.int32, device=DEV), torch.tensor([64], device=DEV))
    want = b.step(tok, seq, pos)
    assert not always
    got = b.step(tok, seq, pos, shared)
    assert len(always) == 2
    live = pos >= 0
    assert _close(got[live], want[live])
    _one_set_of_pages(b, 6, 64)
    assert torch.equal(b.step(tok, seq, pos, shared)[live], got[live])
    assert not _close(b.step(tok, seq, pos)[live], want[live])


def test_step_shares_by_the_reckoning():
    """64 rows behind 4,096 tokens: the call decides by itself."""
    from epure.serving import BatchDecoder
    b = BatchDecoder(_wide(4160), seqs=65, page_size=64)
    _behind_a_prefix(b, 64, (torch.arange(4096) * 37 + 5) % 1000, [1 + i % 7 for i in range(64)])
    seq = torch.arange(64, dtype=torch.int32, device=DEV)
    tok, pos = torch.arange(64, device=DEV) * 13, 4097 + torch.arange(64, device=DEV) % 7
    shared = (torch.tensor([0, 64], dtype=torch.int32, device=DEV), torch.tensor([4096], device=DEV))
    want, got = b.step(tok, seq, pos), b.step(tok, seq, pos, shared)
    assert _close(got, want)
    _one_set_of_pages(b, 64, 4096)
    assert torch.equal(b.step(tok, seq, pos, shared), got)
    assert not _close(b.step(tok, seq, pos), want)


@pytest.mark.parametrize("fmt", ["same", "fp8"])
def test_generate_captured_behind_a_prefix(fmt, always, monkeypatch):
    """The captured steps share too, replay after replay and for a second prefix of another length, and give the eager
    steps' tokens."""
    from epure.serving import BatchDecoder
    b = BatchDecoder(_decoder(), seqs=6, format=fmt, page_size=16)
    free = b.cache.free_pages()
    prompts = _prompts([3, 9, 1, 20, 7])
    begin = b._begin

    def begin_with_one_set(p, n_new, prefix):
        got = begin(p, n_new, prefix)
        _one_set_of_pages(b, len(p), len(prefix))
        return got

    for n in (64, 32):
        prefix = _prompts([n])[0]
        one, two = b.generate(prompts, 6, prefix=prefix), b.generate(prompts, 6, prefix=prefix, graph=False)
        assert torch.equal(one, two)
        with monkeypatch.context() as m:
            m.setattr(b, "_begin", begin_with_one_set)
            assert torch.equal(b.generate(prompts, 6, prefix=prefix), one)
            assert torch.equal(b.generate(prompts, 6, prefix=prefix, graph=False), one)
    assert always and b.cache.free_pages() == free


@pytest.mark.parametrize("fmt", ["same", "int8"])
def test_judge_shares_a_sequence_among_its_drafts(fmt, always):
    """Rows of one sequence on the shared form: the choices of rows by themselves, ragged drafts and an idle row among them,
    eager and in a graph."""
    from epure.serving import BatchDecoder
    b = BatchDecoder(_decoder(), seqs=4, format=fmt, page_size=16)
    lengths, n = [70, 33, 101, 8], 4
    for i, p in enumerate(_prompts(lengths)):
        b.cache.reserve(i, len(p) + n + 1)
        b.prefill(i, p)
    seq = torch.arange(4, dtype=torch.int32, device=DEV)
    tok = torch.tensor([1, 700, 33, 4], device=DEV)
    drafts = (torch.arange(16, device=DEV).view(4, 4) * 61) % 1000
    drafts[2, 2:] = -1
    pos = torch.tensor([70, 33, 101, -1], device=DEV)
    u = torch.rand(4, n + 1, generator=torch.Generator(device=DEV).manual_seed(0), device=DEV)
    # the logits of the same rows, read row by row
    at = torch.where(torch.cat((tok[:, None], drafts), 1) >= 0, pos[:, None] + torch.arange(n + 1, device=DEV), -1)
    at[3] = -1
    rows = (torch.cat((tok[:, None], drafts), 1).clamp(min=0).view(-1), seq.repeat_interleave(n + 1), at.view(-1))
    want = b.step(*rows)
    starts = torch.arange(0, 21, 5, dtype=torch.int32, device=DEV)
    got = b.step(*rows, (starts, (pos + 1).clamp(min=0)))
    live = at.view(-1) >= 0
    assert len(always) == 2 and _close(got[live], want[live])
    one = b.judge(tok, drafts, seq, pos, u, temperature=0.7)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        b.judge(tok, drafts, seq, pos, u, temperature=0.7)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        two = b.judge(tok, drafts, seq, pos, u, temperature=0.7)
    for _ in range(2):
        graph.replay()
        assert torch.equal(one[0][:3], two[0][:3]) and torch.equal(one[1][:3], two[1][:3])


def test_speculate_on_the_shared_form(always):
    from epure.serving import BatchDecoder
    b = BatchDecoder(_decoder(), seqs=3, page_size=16)
    free = b.cache.free_pages()
    prompts = [torch.tensor([5, 6, 7, 8] * 5), torch.tensor([1, 2, 3]), torch.tensor([9])]
    out, passes = b.speculate(prompts, 10, prefix=_prompts([40])[0])
    assert out.shape == (3, 10) and bool((out >= 0).all()) and len(always) == 2 * passes and b.cache.free_pages() == free
