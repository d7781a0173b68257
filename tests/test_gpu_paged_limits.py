"""Attention over a paged cache at the limits of its numbers.  Tolerances are those of ``test_gpu_paged.Batch.check`` unless a test says otherwise."""
import pytest

from tests.test_gpu_paged import BF, Batch, _randn

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("tokens", [1, 50])
@pytest.mark.parametrize("scale", [1e-40, -3e-41, 2e-38])
def test_scales_below_the_smallest_normal_number(scale, tokens, d):
    """Queries and keys of 2^60 bring scores of 2^-10 to 2^-4 even so.  As fp32 such a scale is off by at most 2^-150: 2^-150 times a sum |q k| of 2^127.5
    at most is below 2^-22 of a weight, a quarter of what the tolerance gives it."""
    b = Batch([150, 77], [tokens] * 2, 2, d, 32, BF, 61)
    b.cache.k.mul_(2.0 ** 60)
    q = _randn((b.n, 4, d), 66, BF) * 2.0 ** 60             # not one of the keys, whose product with itself is beyond fp32
    b.check(q, b.attend(q, scale=scale), scale)
