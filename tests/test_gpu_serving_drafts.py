"""Batched decoding behind a common prefix, with drafted tokens and over selected blocks (epure.serving)."""
import pytest
import torch
from test_gpu_serving import DEV, _decoder, _gpu, _prompts  # noqa: F401 (_gpu: a fixture)

pytestmark = pytest.mark.gpu


def _close(a, b, tol=2e-2):
    """Rounding order of linears and attention, as between the other decoders."""
    return float((a - b).abs().max() / b.abs().max()) <= tol


def _wide(max_len, **kw):
    from epure.model import PackedDecoder
    from epure.synthetic import DecoderShapes
    return PackedDecoder(DecoderShapes("qwen3-small", 2, 512, 1024, 16, 4, 128, 1000), device=DEV, seed=3, max_len=max_len, **kw)


@pytest.mark.parametrize("fmt", ["same", "int8"])
def test_step_behind_a_prefix(fmt):
    """24 sequences behind 2,000 tokens that lie in one set of pages: a step that reads them once gives the logits of one
    that reads them for every row (enough for the shared form: 24 rows of 2,000 tokens of 2 KB)."""
    from epure.serving import BatchDecoder
    b = BatchDecoder(_wide(2100), seqs=24, format=fmt, page_size=64)
    prefix = (torch.arange(2000) * 37 + 5) % 1000
    b.cache.reserve(0, 2040)
    b.prefill(0, prefix)
    for i in range(1, 24):
        assert b.cache.share(i, 0, 2000) == 1984
        b.cache.reserve(i, 2040)
        b.prefill(i, prefix[1984:], past=1984)
    for i in range(24):
        b.prefill(i, (torch.arange(1 + i % 7) * 91 + i) % 1000, past=2000)
    tok = torch.arange(24, device=DEV) * 13
    pos = torch.tensor([2001 + i % 7 if i != 5 else -1 for i in range(24)], device=DEV)
    seq = torch.arange(24, dtype=torch.int32, device=DEV)
    want = b.step(tok, seq, pos)
    shared = (torch.tensor([0, 24], dtype=torch.int32, device=DEV), torch.tensor([2000], device=DEV))
    got = b.step(tok, seq, pos, shared)
    live = pos >= 0
    assert _close(got[live], want[live])


@pytest.mark.parametrize("fmt", ["same", "fp8"])
def test_generate_behind_a_prefix(fmt):
    """Graph and eager decoding give the same tokens, the first one is the prompts' with the prefix written out, the prefix's
    pages are held once, and all pages come back."""
    from epure.serving import BatchDecoder
    b = BatchDecoder(_decoder(), seqs=5, format=fmt, page_size=16)
    free = b.cache.free_pages()
    prefix, prompts = _prompts([50])[0], _prompts([3, 9, 1, 20, 7])
    one = b.generate(prompts, 6, prefix=prefix)
    two = b.generate(prompts, 6, prefix=prefix, graph=False)
    assert torch.equal(one, two) and one.shape == (5, 6) and b.cache.free_pages() == free
    assert torch.equal(b.generate(prompts, 6, prefix=prefix), one)
    b._begin(prompts, 6, prefix)
    # 48 tokens of the prefix in three pages for all; each sequence's rest: 2 of the prefix, its prompt and 6 more
    assert free - b.cache.free_pages() == 3 + sum(-(-(2 + len(p) + 6) // 16) for p in prompts)
    for i in range(5):
        b.cache.release(i)
    for i, p in enumerate(prompts):
        whole = b.prefill(0, torch.cat((prefix, p)))
        b.cache.release(0)
        b.prefill(0, prefix)
        assert _close(b.prefill(0, p, past=50), whole, 2e-2 if fmt == "same" else 1e-1)
        b.cache.release(0)
    assert b.cache.free_pages() == free


@pytest.mark.parametrize("fmt", ["same", "int8"])
def test_judge_agrees_with_single_steps(fmt):
    """Drafts are kept as long as they are what single steps would take (temperature 0), ragged ones and an idle row among
    them, and the token behind them is the steps' too; places where two tokens are within rounding of each other say
    nothing."""
    from epure.serving import BatchDecoder
    b = BatchDecoder(_decoder(), seqs=4, format=fmt, page_size=16)
    prompts = _prompts([5, 30, 17, 8])
    n = 4
    first = []
    for i, p in enumerate(prompts):
        b.cache.reserve(i, len(p) + n + 2)
        first.append(int(b.prefill(i, p).argmax()))
    seq = torch.arange(4, dtype=torch.int32, device=DEV)
    at = [len(p) for p in prompts]
    greedy, gaps = [[t] for t in first], [[] for _ in range(4)]
    for s in range(n + 1):
        logits = b.step(torch.tensor([g[-1] for g in greedy], device=DEV), seq, torch.tensor(at, device=DEV) + s)
        top = logits.topk(2, -1).values
        for i in range(4):
            greedy[i].append(int(logits[i].argmax()))
            gaps[i].append(float((top[i, 0] - top[i, 1]) / logits[i].abs().max()))
    drafts = torch.tensor([g[1:1 + n] for g in greedy])
    drafts[1, 2] = (drafts[1, 2] + 1) % 1000               # a wrong one
    drafts[2, 3] = -1                                      # three drafts
    pos = torch.tensor([at[0], at[1], at[2], -1], device=DEV)
    u = torch.rand(4, n + 1, generator=torch.Generator(device=DEV).manual_seed(0), device=DEV)
    got, kept = b.judge(torch.tensor(first, device=DEV), drafts.to(DEV), seq, pos, u, temperature=0.0)
    for i, k in ((0, 4), (1, 2), (2, 3)):
        if min(gaps[i][:k + 1]) > 2e-2:
            assert int(kept[i]) == k
            assert got[i].tolist() == greedy[i][1:k + 2] + [-1] * (n - k)
    # with a temperature: from the target's own probabilities, with a draft model's
    probs = torch.softmax(torch.randn(4, n, 1000, generator=torch.Generator(device=DEV).manual_seed(1), device=DEV), -1)
    got, kept = b.judge(torch.tensor(first, device=DEV), drafts.clamp(min=0).to(DEV), seq, pos, u, temperature=0.7,
                        draft_probs=probs)
    assert bool((kept >= 0).all()) and bool((got[:3, 0] >= 0).all())


def test_judge_ends_at_a_draft_outside_the_vocabulary():
    """Such a draft is not looked up in the embedding: the row is judged as one that ends there."""
    from epure.serving import BatchDecoder
    b = BatchDecoder(_decoder(), seqs=2, page_size=16)
    prompts = _prompts([5, 9])
    for i, p in enumerate(prompts):
        b.cache.reserve(i, len(p) + 4)
        b.prefill(i, p)
    seq, pos = torch.arange(2, dtype=torch.int32, device=DEV), torch.tensor([5, 9], device=DEV)
    tok, u = torch.tensor([1, 2], device=DEV), torch.full((2, 4), 0.25, device=DEV)
    want = b.judge(tok, torch.tensor([[3, -1, -1], [-1, 4, 4]], device=DEV), seq, pos, u, temperature=1.0)
    for bad in (1000, 2 ** 40):
        got = b.judge(tok, torch.tensor([[3, bad, 4], [bad, 4, 4]], device=DEV), seq, pos, u, temperature=1.0)
        for x, y in zip(got, want):
            assert torch.equal(x, y)


def test_judge_behind_long_sequences():
    """Drafts of sequences long enough for the shared form: the logits' choice equals that of rows by themselves."""
    from epure.serving import BatchDecoder
    b = BatchDecoder(_wide(2100), seqs=6, format="same", page_size=64)
    for i in range(6):
        b.cache.reserve(i, 2020)
        b.prefill(i, (torch.arange(1990 + i) * 37 + i) % 1000)
    seq = torch.arange(6, dtype=torch.int32, device=DEV).repeat_interleave(8)
    pos = (1990 + torch.arange(6, device=DEV))[:, None] + torch.arange(8, device=DEV)
    tok = (torch.arange(48, device=DEV) * 17) % 1000
    want = b.step(tok, seq, pos.reshape(-1))
    starts = torch.arange(0, 49, 8, dtype=torch.int32, device=DEV)
    got = b.step(tok, seq, pos.reshape(-1), (starts, pos[:, 0] + 1))
    assert _close(got, want)


@pytest.mark.parametrize("kw", [dict(), dict(temperature=0.8), dict(drafts=0), dict(prefix=True, drafts=2)])
def test_speculate(kw):
    from epure.serving import BatchDecoder
    b = BatchDecoder(_decoder(), seqs=3, format="int8", page_size=16)
    free = b.cache.free_pages()
    prompts = [torch.tensor([5, 6, 7, 8] * 5), torch.tensor([1, 2, 3]), torch.tensor([9])]
    if kw.pop("prefix", False):
        kw["prefix"] = _prompts([20])[0]
    gen = torch.Generator(device=DEV).manual_seed(4)
    out, passes = b.speculate(prompts, 10, generator=gen, **kw)
    assert out.shape == (3, 10) and bool((out >= 0).all()) and bool((out < 1000).all()) and 1 <= passes <= 10
    assert b.cache.free_pages() == free


def test_speculate_draws_its_first_token_too():
    """With a temperature the token behind each prompt is drawn like the others, not the most likely one."""
    from epure import sampling
    from epure.serving import BatchDecoder
    b = BatchDecoder(_decoder(), seqs=3, page_size=16)
    prompts = _prompts([5, 9, 17])
    logits = []
    for i, p in enumerate(prompts):
        b.cache.reserve(i, len(p))
        logits.append(b.prefill(i, p))
        b.cache.release(i)
    logits = torch.stack(logits)
    u = torch.rand(3, 1, device=DEV, generator=torch.Generator(device=DEV).manual_seed(8))
    want, _ = sampling.verify(torch.softmax(logits / 5.0, -1)[:, None], None, torch.empty(3, 0, dtype=torch.long, device=DEV), u)
    got, _ = b.speculate(prompts, 1, temperature=5.0, generator=torch.Generator(device=DEV).manual_seed(8))
    assert torch.equal(got, want)
    assert not torch.equal(got[:, 0], logits.argmax(-1))


def test_speculate_no_or_one_token():
    """Nothing to generate, and the token that the prompts themselves give."""
    from epure.serving import BatchDecoder
    b = BatchDecoder(_decoder(), seqs=2, page_size=16)
    prompts = _prompts([5, 9])
    got, passes = b.speculate(prompts, 0)
    assert got.shape == (2, 0) and got.dtype == torch.long and passes == 0
    got, passes = b.speculate(prompts, 1)
    assert got.shape == (2, 1) and passes == 0
    assert torch.equal(got, b.generate(prompts, 1))


@pytest.mark.parametrize("fmt", ["same", "int8", "fp8"])
def test_sparse_steps(fmt):
    """A selection that covers every block gives the dense steps' logits; a small one runs, in a graph as well, and its bounds
    are those of the pages."""
    from epure import paged
    from epure.serving import BatchDecoder
    dec = _decoder()
    dense, all_of_it = BatchDecoder(dec, seqs=3, format=fmt, page_size=16), BatchDecoder(dec, seqs=3, format=fmt, page_size=16,
                                                                                         sparse=(8, 1, 1))
    prompts = _prompts([5, 90, 33])
    seq, tok = torch.arange(3, dtype=torch.int32, device=DEV), torch.tensor([7, 300, 999], device=DEV)
    for b in (dense, all_of_it):
        for i, p in enumerate(prompts):
            b.cache.reserve(i, len(p) + 4)
            b.prefill(i, p)
    for t in range(3):
        pos = torch.tensor([len(p) + t for p in prompts], device=DEV)
        assert _close(all_of_it.step(tok - t, seq, pos), dense.step(tok - t, seq, pos))
    pages = all_of_it.cache.layer(1)
    for i, p in enumerate(prompts):
        n = len(p) + 3
        for j in range(-(-n // 16)):
            at = torch.arange(16 * j, min(n, 16 * j + 16), device=DEV)
            k, _ = paged.read(pages, torch.full_like(at, i, dtype=torch.int32), at, torch.float32 if fmt != "same" else None)
            got = all_of_it.cache.bounds[1, int(pages.table[i, j])]
            assert torch.equal(got, torch.stack((k.amin(0), k.amax(0)), 1).to(torch.bfloat16))
    few = BatchDecoder(dec, seqs=3, format=fmt, page_size=16, sparse=(3, 1, 1))
    assert torch.equal(few.generate(prompts, 6), few.generate(prompts, 6, graph=False))
    assert few.generate(prompts, 6, prefix=_prompts([20])[0]).shape == (3, 6)


def test_refusals():
    from epure.serving import BatchDecoder
    dec = _decoder()
    for bad in ((0, 0, 0), (2, 2, 1), (3, -1, 1)):
        with pytest.raises(ValueError, match="sparse"):
            BatchDecoder(dec, sparse=bad)
    b = BatchDecoder(dec, seqs=2, page_size=16, sparse=(3, 1, 1))
    z = torch.zeros(2, dtype=torch.long, device=DEV)
    with pytest.raises(ValueError, match="whole cache"):
        b.judge(z, z.view(2, 1), z.int(), z, torch.zeros(2, 2, device=DEV))
    with pytest.raises(ValueError, match="shared prefix"):
        b.step(z, z.int(), z, (z.int(), z[:1]))
    b.cache.reserve(0, 20)
    free = b.cache.free_pages()
    for call in (b.speculate, b.generate):
        with pytest.raises(ValueError):
            call(_prompts([3, 3, 3]), 2)
    assert b.cache.free_pages() == free                    # what the caller holds stays
