"""Attention over a 4-bit cache where the order of magnitude of what it multiplies decides: sums that cancel, rows that a query does not see
and that hold anything, weights next to nothing, and large scores over many rows.  Tolerances are derived at each test."""
import pytest
import torch

from oracle import int4_oracle as O
from tests.gpu_util import DEV, assert_clean_device
from tests.test_gpu_int4 import BF, HF, _cache, _check_attention, _d, _randn

pytestmark = pytest.mark.gpu


def _held(x, dtype):
    """Rows ``x [B, H, L, D]`` as the cache holds them: codes, scales, and the values in 64 bits."""
    codes, s = O.quantize(x.to(dtype), 64)
    return O.pack(codes).to(DEV), s.to(dtype).to(DEV), O.values(codes, s, 64).to(DEV)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("d,rows", [(64, 256), (128, 301), (256, 64)])
def test_weights_that_cancel(d, rows, dtype):
    """Values of +1 and -1 under weights that differ by little: the result is the difference, of which a rounding of the weights to 11 bits would
    leave two or three.  A weight is off by 2^-22 (exponential) and 2^-22 (two fp16 numbers) of itself, the scores being below 1/2 by 2^-23;
    sums over the rows by one step in 2^23 for every 16, 301 / 16 of them, in the total and in the result, and for joining warps: below 2^-17 of
    sum p |v| = 1 together."""
    k, v = torch.zeros((1, 1, rows, d)), torch.ones((1, 1, rows, d))
    k[..., 1::2, 0] = -1.0
    v[..., 1::2, :] = -1.0
    kc, ks, kv = _held(k, dtype)
    vc, vs, vv = _held(v, dtype)
    a = torch.logspace(-2.5, -0.4, 21)
    q = torch.zeros((1, 1, 21, d))
    q[0, 0, :, 0] = a
    q = q.to(dtype).to(DEV)
    n = rows + 20                                           # every query sees all rows: lengths beyond the cache end with it
    got = _d().attention_int4_cache(q, _d().Int4KVCache(kc, ks, vc, vs), torch.tensor([n], device=DEV), scale=1.0)
    want = O.attention(q, kv, vv, [n], scale=1.0)
    tol = want.abs() * (torch.finfo(dtype).eps / 2) * (1 + 2 ** -8) + 2.0 ** -17
    err = (got.double() - want).abs()
    assert bool((err <= tol).all()), (err / tol).max().item()
    assert_clean_device()
