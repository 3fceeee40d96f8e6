"""Precision of the paged attention's weights: small ones beside a peak, and the two parts of 16-bit ones."""
import math

import pytest
import torch
from test_gpu_paged import DEV, UNIT, _fill, _gen, _gpu, _pages, _reference, _tokens  # noqa: F401 (_gpu: a fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fmt", ["same", "int8", "fp8"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n,peak", [(64, 0), (160, 0), (160, 159), (160, 80)])
def test_many_small_weights_beside_a_peak(fmt, dtype, n, peak):
    """One token 17.5 nats above n - 1 others, whose values lie in another dim: their weights, each 2^-25.2 of the
    largest, must not vanish from the numerator.

    A weight in f16 is carried 2^7 above the maximum's 1, and f16's smallest step is 2^-24: each of the others is
    off by at most 2^-25 - 7 of the largest.  Besides: the result's rounding, one of a weight of a warp that has
    no peak (2^-11), the key's 8-bit row (17.5 off by a few 2^-24) and 2^-18 of exp2 and the sums."""
    from epure import paged
    pages = _pages([n], 1, 64, 16, fmt, dtype)
    seq, pos = _tokens([n])
    k, v = torch.zeros(n, 1, 64, device=DEV, dtype=dtype), torch.zeros(n, 1, 64, device=DEV, dtype=dtype)
    k[peak, 0, 0] = 17.5
    v[:, 0, 1] = 64
    v[peak, 0, 0], v[peak, 0, 1] = 64, 0
    paged.write(pages, k, v, seq, pos)
    q = torch.zeros(1, 4, 64, device=DEV, dtype=dtype)
    q[..., 0] = 1
    out, lse = paged.attend(pages, q, torch.tensor([n], device=DEV), scale=1.0, return_lse=True)
    total = 1 + (n - 1) * math.exp(-17.5)
    want = 64 * (n - 1) * math.exp(-17.5) / total
    bound = want * (UNIT[dtype] + 2.0 ** -11 + 2.0 ** -17) + 64 * (n - 1) * 2.0 ** -32
    assert float((out[..., 1].double() - want).abs().max()) <= bound
    assert float((out[..., 0].double() - 64 / total).abs().max()) <= 64 * (UNIT[dtype] + 2.0 ** -11)
    assert float((lse.double() - 17.5 - math.log(total)).abs().max()) <= 2.0 ** -18


@pytest.mark.parametrize("fmt", ["same", "int8", "fp8"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_weights_are_held_in_two_parts(fmt, dtype):
    """Values of +-1 whose weighted sums cancel: one rounding of a weight to 16 bits would show.

    Bounds: a weight is two values of the tensor cores' type, so it is off by its unit roundoff squared (bf16 for
    bf16 caches, else f16); twice its score's error (numerator and sum) and 2^-18 of exp2, log2 and the sums; all
    of the weighted |v|; the result's rounding (2^-25: f16's smallest step)."""
    from epure import paged
    lengths = [5 + i % 8 for i in range(64)]
    pages = _pages(lengths, 1, 16, 16, fmt, dtype)
    seq, pos = _tokens(lengths)
    g = _gen(31)
    k = (torch.rand(len(pos), 1, 16, generator=g, device=DEV) - 0.5).to(dtype)
    v = (torch.randint(0, 2, (len(pos), 1, 16), generator=g, device=DEV) * 2 - 1).to(dtype)
    paged.write(pages, k, v, seq, pos)
    if fmt != "same":
        k, v = paged.read(pages, seq, pos, torch.float32)
    q = torch.randn(64, 8, 16, generator=g, device=DEV).to(dtype)
    out = paged.attend(pages, q, torch.tensor(lengths, device=DEV))
    want, _, mag, err = _reference(q, k.double(), v.double(), lengths, 0, 0.25)
    unit = UNIT[dtype if fmt == "same" else torch.float16]
    bound = UNIT[dtype] * want.abs() + (unit ** 2 + 2 * err[..., None] + 2.0 ** -18) * 1.01 * mag + 2.0 ** -25
    off = (out.double() - want).abs()
    assert bool((off <= bound).all()), (float((off / bound).max()), int((off > bound).sum()))
