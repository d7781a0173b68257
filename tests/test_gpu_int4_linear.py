"""``BlockInt4Linear`` in a program: checkpoints after the first forward, types of model and activations."""
import pytest
import torch

from tests.gpu_util import DEV, assert_clean_device, set_config
from tests.test_gpu_int4 import BF, HF, _f, _randn

pytestmark = pytest.mark.gpu


def _layer(dtype=BF, seed=1, k=200, n=130):
    from blockwise_int8_linear_b200 import BlockInt4Linear
    m = BlockInt4Linear(k, n, device=DEV, dtype=dtype).eval()
    m.weight.data, m.bias.data = _randn((n, k), seed, dtype, 0.05), _randn((n,), seed + 1, dtype)
    return m


@pytest.mark.parametrize("drop", [False, True])
def test_loading_another_weight_after_the_first_forward(drop):
    """The next forward is that of a new layer with the weight, not that of the codes from before."""
    set_config(64, BF)
    x = _randn((3, 200), 9, BF)
    a, b = _layer(seed=1), _layer(seed=5)
    floating = {k: v.clone() for k, v in b.state_dict().items()}
    a(x)
    a.prepare_for_eval(drop_weight=drop)
    a.load_state_dict(floating)
    assert torch.equal(a(x), b(x))
    half = _layer(HF, seed=7)
    set_config(64, HF)
    half(x.to(HF))
    a.load_state_dict(half.state_dict())
    # parameters are copied into the layer's type, as nn.Linear's are: the bias is half's in bf16
    assert torch.equal(a(x.to(HF)), _f().int4_matmul(x.to(HF), half.W_int4, half.state_W4, half.bias.detach().to(BF)))
    set_config(64, BF)
    assert_clean_device()
