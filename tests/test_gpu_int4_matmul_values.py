"""The 4-bit matrix product over the whole range of its activations, in batches of every size, and at offsets beyond 32 bits."""
import pytest
import torch

from tests.gpu_util import DEV, assert_clean_device
from tests.test_gpu_int4 import BF, FF, HF, _check_product, _f, _randn, _weights

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


@pytest.mark.parametrize("dtype", [BF, HF])
def test_a_row_alone_and_among_others(dtype):
    """A row's result in batches of 1 to 70 rows, whose divisions of the work differ: each within the tolerance, and a call repeated gives its bits."""
    f = _f()
    codes, state, w = _weights(130, 1200, 64, dtype, 2)
    x = _randn((70, 1200), 3, dtype, 1.0, outliers=0.01)
    for m in (1, 2, 8, 9, 16, 17, 33, 64, 65, 70):
        y = f.int4_matmul(x[:m], codes, state, fblock_size=64, dtype=FF)
        _check_product(y, x[:m], w, state, 64)
        assert torch.equal(f.int4_matmul(x[:m], codes, state, fblock_size=64, dtype=FF), y)
    assert_clean_device()


def test_more_than_2_to_the_31_bytes():
    """Codes of a weight, and a matrix that is quantized and read back, whose offsets pass 32 bits: the last rows are those of the same rows alone."""
    f = _f()
    k, n = 65536, 65600                                     # 2.15e9 bytes of codes
    g = torch.Generator(device=DEV).manual_seed(1)
    codes = torch.randint(0x11, 0x100, (n, k // 2), dtype=torch.uint8, device=DEV, generator=g)
    state = (torch.rand((n, k // 128), device=DEV, generator=g) * 0.01).to(BF)
    x = _randn((3, k), 3, BF)
    y = f.int4_matmul(x, codes, state, fblock_size=128, dtype=FF)
    last = slice(n - 40, n)
    q = torch.stack((codes[last] & 15, codes[last] >> 4), -1).flatten(-2).double() - 8
    _check_product(y[:, last], x, q * state[last].double().repeat_interleave(128, -1) / 7, state[last], 128)
    v = f.dequantize_block_int4(codes, state, 128, dtype=BF)
    assert torch.equal(v[last], f.dequantize_block_int4(codes[last].clone(), state[last].clone(), 128, dtype=BF))
    del codes, state, y
    codes, state = f.quantize_block_int4(v, 64)             # 4.3e9 values
    for part in (last, slice(0, 8), slice(32760, 32776)):
        c, s = f.quantize_block_int4(v[part].clone(), 64)
        assert torch.equal(codes[part], c) and torch.equal(state[part], s)
    assert_clean_device()
