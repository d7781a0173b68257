"""``BlockInt4Linear`` in a program: checkpoints after the first forward, types of model and activations."""
import pytest
import torch

from tests.gpu_util import DEV, assert_clean_device, set_config
from tests.test_gpu_int4 import BF, FF, HF, _f, _randn

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


def test_types_of_model_and_activations():
    """A chain of layers runs in a float32 model, an fp16 model under results in bf16, and after a cast of the model; results are the functional
    product's on activations in the scales' type."""
    f = _f()

    def chain(dtype, out):
        set_config(64, out)
        net = torch.nn.Sequential(_layer(dtype, 1, 200, 130), _layer(dtype, 3, 130, 64)).eval()
        return net, _randn((5, 200), 9, dtype)

    def want(net, x):
        for m in net:
            x = f.int4_matmul(x.to(m.state_W4.dtype), m.W_int4, m.state_W4, m.bias.detach())
        return x

    for dtype, out in ((FF, BF), (FF, HF), (FF, FF), (HF, BF), (HF, FF), (BF, FF), (BF, BF), (HF, HF)):
        net, x = chain(dtype, out)
        y = net(x)
        assert y.dtype == out and torch.equal(y, want(net, x))
        state = [m.state_W4.clone() for m in net]
        net.float()
        assert all(torch.equal(m.state_W4, s) and m.state_W4.dtype == s.dtype for m, s in zip(net, state))
        got = net(x.float())
        assert torch.equal(got, want(net, x.float()))
    net, x = chain(HF, BF)
    assert bool(net[0](torch.full((1, 200), 1e5, dtype=BF, device=DEV)).isfinite().logical_not().all())      # loudly, beyond fp16
    net, x = chain(BF, BF)
    with pytest.raises(ValueError, match="one type"):
        net(x.to(HF))
    assert_clean_device()
