"""The 4-bit quantizer's arithmetic for every scale: 8 significant bits (bf16) and 11 (fp16)."""
import numpy as np
import pytest

from tests.test_int4_host import _codes_as_the_kernel

F32 = np.float32


@pytest.mark.parametrize("off", [-1, 0, 1])
@pytest.mark.parametrize("bits", [8, 11])
def test_every_scale_and_every_value_below_it(bits, off):
    """rint(7 x / s), ties to even, decided by integers, for all significands of scale and value and the six exponents of a value in which a
    code is not 0, with a reciprocal that is the nearest one or a step beside it."""
    m = np.arange(1 << (bits - 1), 1 << bits, dtype=np.int64)
    s = m[:, None]
    for e in range(6):                                     # s and x = m 2^-e as multiples of 2^-e
        num, den = 7 * m[None], s << e
        q, rest = num // den, num % den
        q = q + ((2 * rest > den) | ((2 * rest == den) & (q % 2 == 1)))
        x = np.broadcast_to(m[None].astype(F32) * F32(2.0 ** -e), q.shape)
        below = (x <= s) & (q <= 7)
        scale = np.broadcast_to(s, q.shape).astype(F32)
        for sign in (1, -1):
            got = _codes_as_the_kernel(F32(sign) * x, scale, off)
            assert np.array_equal(got[below], sign * q[below])
        assert bool(below.all() if e else below[np.tril_indices(len(m))].all())
