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
