"""Calls of the 4-bit operators that their Python functions refuse, one reason a test."""
import pytest
import torch

from tests.gpu_util import DEV, assert_clean_device
from tests.test_gpu_int4 import BF, HF, _d, _f, _randn, _table, _weights

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("scale", [float("nan"), float("inf"), -float("inf"), 1e39, -1e300])
def test_attention_refuses_a_scale_that_is_no_finite_number(scale):
    o = _d()
    cache = o.int4_kv_cache(1, 1, 16, 64, BF, DEV)
    with pytest.raises(ValueError, match="scale"):
        o.attention_int4_cache(_randn((1, 1, 1, 64), 1, BF), cache, torch.tensor([3], device=DEV), scale=scale)
    assert_clean_device()


def _calls():
    """Every operator as a function of its floating-point operands, by name."""
    f, o = _f(), _d()
    codes, state, _ = _weights(32, 128, 64, BF, 1)
    cache = o.int4_kv_cache(2, 2, 16, 64, BF, DEV)
    n = torch.tensor([3], device=DEV)
    with_states = lambda k, v: cache._replace(k_state=k, v_state=v)
    return {
        "quantize": (lambda x: f.quantize_block_int4(x, 64), {"x": _randn((2, 128), 1, BF)}),
        "dequantize": (lambda state: f.dequantize_block_int4(codes, state, 64), {"state": state}),
        "matmul": (lambda x, state, bias, residual: f.int4_matmul(x, codes, state, bias, residual=residual, fblock_size=64, dtype=BF),
                   {"x": _randn((2, 128), 1, BF), "state": state, "bias": _randn((32,), 2, BF), "residual": _randn((2, 32), 3, BF)}),
        "append": (lambda qkv, cis, k, v: o.rope_cache_append_int4(qkv, cis, n, with_states(k, v)),
                   {"qkv": _randn((2, 1, 8, 64), 1, BF), "cis": torch.view_as_real(_table(16, 64)).clone(), "k": cache.k_state, "v": cache.v_state}),
        "attention": (lambda q, k, v: o.attention_int4_cache(q, with_states(k, v), n),
                      {"q": _randn((2, 4, 1, 64), 1, BF), "k": cache.k_state, "v": cache.v_state}),
    }


@pytest.mark.parametrize("name", ["quantize", "dequantize", "matmul", "append", "attention"])
def test_no_derivative_is_lost_silently(name):
    """Each floating-point operand in turn wants a gradient, or brings a tangent: refused, but for the former under no_grad."""
    import torch.autograd.forward_ad as fwd
    call, operands = _calls()[name]
    want = call(**operands)
    want = want if isinstance(want, tuple) else (want,)
    for at, x in operands.items():
        wants = {**operands, at: x.clone().requires_grad_(True)}
        with pytest.raises(RuntimeError, match="backward"):
            call(**wants)
        with torch.no_grad():
            got = call(**wants)
        assert all(torch.equal(a, b) for a, b in zip(got if isinstance(got, tuple) else (got,), want))
        with fwd.dual_level():
            dual = {**operands, at: fwd.make_dual(x.clone(), torch.ones_like(x))}
            with pytest.raises(RuntimeError, match="tangent"):
                call(**dual)
            with torch.no_grad(), pytest.raises(RuntimeError, match="tangent"):
                call(**dual)
    assert_clean_device()
