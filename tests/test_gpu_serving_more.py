"""Batched decoding: a sequence's logits do not depend on what its neighbours hold; batches of every size."""
import pytest
import torch
from test_gpu_serving import DEV, TOLERANCE, _decoder, _gpu, _prompts  # noqa: F401 (_gpu: a fixture)

pytestmark = pytest.mark.gpu


def _steps(dec, fmt, prompts, feed):
    """Logits [steps, batch, vocab] after the prompts and teacher-forced tokens feed [steps, batch]."""
    from epure.serving import BatchDecoder
    b = BatchDecoder(dec, seqs=len(prompts), format=fmt, page_size=16)
    for i, p in enumerate(prompts):
        b.prefill(i, p)
        b.cache.reserve(i, len(p) + len(feed))
    seq = torch.arange(len(prompts), dtype=torch.int32, device=DEV)
    start = torch.tensor([len(p) for p in prompts], device=DEV)
    return torch.stack([b.step(f.to(DEV), seq, start + t) for t, f in enumerate(feed)])


@pytest.mark.parametrize("fmt", ["same", "int8", "fp8"])
@pytest.mark.parametrize("hidden,batch", [(512, 5), (2048, 24)])
def test_neighbours(fmt, hidden, batch):
    """Other tokens in the neighbours, of the same number, change nothing: not a bit.  Alone, the sequence takes
    other shapes of the linears and another plan of the attention, which round in another order."""
    dec = _decoder(hidden=hidden)
    lengths = [3 + 5 * (i % 7) for i in range(batch)]
    prompts, feed = _prompts(lengths), (torch.arange(3 * batch).view(3, batch) * 53) % 1000
    got = _steps(dec, fmt, prompts, feed)
    mine = batch // 2
    others = [p if i == mine else (p * 7 + 13) % 1000 for i, p in enumerate(prompts)]
    other_feed = (feed * 3 + 1) % 1000
    other_feed[:, mine] = feed[:, mine]
    again = _steps(dec, fmt, others, other_feed)
    assert torch.equal(again[:, mine], got[:, mine])
    assert not torch.equal(again[:, 0], got[:, 0])
    alone = _steps(dec, fmt, [prompts[mine]], feed[:, mine:mine + 1])[:, 0]
    assert float((alone - got[:, mine]).abs().max() / alone.abs().max()) <= TOLERANCE[fmt]


def test_rotation_has_the_tensor_formulas_gradient_bit_for_bit():
    """epure.rotary.rope against autograd of the rotation in tensor operations (float32 inside, one rounding)."""
    from epure import rotary
    g = torch.Generator(device=DEV).manual_seed(61)
    cos, sin = rotary.rope_tables(64, 100, DEV)
    pos = torch.randint(0, 100, (50,), generator=g, device=DEV)
    q, k, dq, dk = (torch.randn(50, h, 64, generator=g, device=DEV).to(torch.bfloat16) for h in (6, 2, 6, 2))

    def formula(x):
        c, s = cos[pos][:, None], sin[pos][:, None]
        a, b = x.float()[..., :32], x.float()[..., 32:]
        return torch.cat([a * c - b * s, b * c + a * s], -1).to(x.dtype)

    q, k = q.requires_grad_(True), k.requires_grad_(True)
    want = torch.autograd.grad((formula(q), formula(k)), (q, k), (dq, dk))
    got = torch.autograd.grad(rotary.rope(q, k, pos, cos, sin), (q, k), (dq, dk))
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("hidden,batch", [(512, 11), (512, 12), (512, 16), (2048, 8), (2048, 9), (2048, 16), (2048, 17)])
def test_batches_around_the_fused_limit(hidden, batch):
    """The fused linears take 8 rows of 2048 features or 11 of 512; larger batches step all the same."""
    dec = _decoder(hidden=hidden)
    lengths = [2 + 3 * (i % 5) for i in range(batch)]
    prompts, feed = _prompts(lengths), (torch.arange(2 * batch).view(2, batch) * 53) % 1000
    got = _steps(dec, "same", prompts, feed)
    f32 = dec.share_weights("fp32")
    for i in (0, batch // 2, batch - 1):
        f32.prefill(prompts[i])
        for t in range(2):
            want = f32.step(feed[t, i:i + 1].to(DEV), torch.tensor([lengths[i] + t], device=DEV))
            assert float((got[t, i] - want).abs().max() / want.abs().max()) <= TOLERANCE["same"]


@pytest.mark.parametrize("k", [512, 2048])
def test_most_rows_of_the_fused_linears(k):
    """What decode_linear_max_rows says is taken, and one row more is refused."""
    from epure import _native, synthetic
    st = [synthetic.make_store(64, k, device=torch.device(DEV), seed=s, gpu_layout="mma16") for s in (1, 2)]
    for epilogue, stores in ((_native.EPI_STORE, st), (_native.EPI_SILU_MUL, st)):
        rows = _native.decode_linear_max_rows(k, _native.PRO_RMSNORM, epilogue)
        assert 1 <= rows <= 16
        x = torch.randn(16, k, device=DEV).to(torch.bfloat16)
        got = _native.decode_linear(x[:rows], stores, prologue=_native.PRO_RMSNORM, epilogue=epilogue)
        one = _native.decode_linear(x[:1], stores, prologue=_native.PRO_RMSNORM, epilogue=epilogue)
        for a, b in zip(got, one):
            assert float((a[0] - b[0]).abs().max()) <= 2.0 ** -7 * float(b.abs().max())
        if rows < 16:
            with pytest.raises(RuntimeError, match=f"at most {rows} "):
                _native.decode_linear(x[:rows + 1], stores, prologue=_native.PRO_RMSNORM, epilogue=epilogue)


def test_idle_rows_at_any_negative_position():
    """They are no error, and leave the other rows as they are."""
    from epure import _native
    from epure.serving import BatchDecoder
    b = BatchDecoder(_decoder(), seqs=3, format="int8", page_size=16)
    b.prefill(1, _prompts([5])[0])
    b.cache.reserve(1, 6)
    tok, seq = torch.tensor([3, 4, 5], device=DEV), torch.arange(3, dtype=torch.int32, device=DEV)
    want = b.step(tok, seq, torch.tensor([-1, 5, -1], device=DEV))
    got = b.step(tok, seq, torch.tensor([-4, 5, -2 ** 40], device=DEV))
    assert _native.device_error() == 0
    assert torch.equal(got, want) and torch.isfinite(got).all()
