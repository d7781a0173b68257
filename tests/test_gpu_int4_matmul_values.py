"""The 4-bit matrix product over the whole range of its activations."""
import pytest
import torch

from tests.gpu_util import DEV, assert_clean_device
from tests.test_gpu_int4 import BF, FF, _check_product, _f, _randn, _weights

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("block", [32, 64, 128])
@pytest.mark.parametrize("m", [1, 8, 16, 32, 64])
def test_activations_up_to_the_largest_number(m, block):
    """Every product of a block has the same sign and x is the largest bf16 number or half of it: the sum of codes times x, 7 * 128 x, is beyond
    fp32, the result is not.  At the other end, x of 1e-36: the tolerance is that of fp32 sums all the same."""
    f = _f()
    k, n = 512, 48
    codes, state, w = _weights(n, k, block, BF, 3, 1e-6)
    big = torch.finfo(BF).max
    x = torch.where(torch.arange(m)[:, None] % 2 == 0, big, big / 2).expand(m, k).to(BF).to(DEV)
    x = x * torch.sign(w[torch.arange(m) % n]).to(BF).to(DEV)       # a row of x has the signs of a row of W
    y = f.int4_matmul(x, codes, state, fblock_size=block, dtype=FF)
    assert bool(y.isfinite().all()) and float(y.max()) > 1e34
    _check_product(y, x, w, state, block)
    codes, state, w = _weights(n, k, block, BF, 4, 1.0)
    small = _randn((m, k), 5, BF, 1e-36)
    _check_product(f.int4_matmul(small, codes, state, fblock_size=block, dtype=FF), small, w, state, block)
    assert_clean_device()
