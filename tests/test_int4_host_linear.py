"""Checkpoints of ``BlockInt4Linear`` on the CPU: which buffers a layer has after loading, and what it refuses to load."""
import pytest
import torch
import torch.nn as nn

from blockwise_int8_linear_b200 import BlockInt4Linear
from oracle import int4_oracle as O


def _quantized(seed=0, dtype=torch.bfloat16, block=64, drop=False, shape=(16, 130)):
    """A layer as the first forward leaves it (the quantizer itself needs a GPU)."""
    m = BlockInt4Linear(shape[1], shape[0], dtype=dtype).eval()
    m.weight.data = torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype)
    q, s = O.quantize(m.weight.detach(), block)
    m.register_buffer("W_int4", O.pack(q))
    m.register_buffer("state_W4", s.to(dtype))
    if drop:
        m.weight.data = torch.empty(0, dtype=dtype)
    return m


@pytest.mark.parametrize("strict", [False, True])
@pytest.mark.parametrize("drop", [False, True])
def test_a_floating_point_weight_drops_what_was_quantized_before(strict, drop):
    m = _quantized(0, drop=drop)
    other = nn.Linear(130, 16, dtype=torch.bfloat16)
    m.load_state_dict(other.state_dict(), strict=strict)
    assert not hasattr(m, "W_int4") and not hasattr(m, "state_W4") and torch.equal(m.weight, other.weight)
    assert set(m.state_dict()) == {"weight", "bias"}


@pytest.mark.parametrize("drop", [False, True])
@pytest.mark.parametrize("dtype,block", [(torch.float16, 64), (torch.bfloat16, 32), (torch.float16, 128)])
def test_buffers_come_as_the_checkpoint_has_them(dtype, block, drop):
    m, other = _quantized(0), _quantized(1, dtype, block, drop)
    m.load_state_dict(other.state_dict())
    assert m.state_W4.dtype == dtype and torch.equal(m.state_W4, other.state_W4) and torch.equal(m.W_int4, other.W_int4)
    assert m.weight.numel() == (0 if drop else 16 * 130)
    fresh = BlockInt4Linear(130, 16).eval()
    fresh.load_state_dict(other.state_dict())
    assert torch.equal(fresh.state_W4, other.state_W4) and torch.equal(fresh.W_int4, other.W_int4)


def test_what_does_not_fit_is_refused():
    m = _quantized(0)
    before = {k: v.clone() for k, v in m.state_dict().items()}
    half = {k: v for k, v in _quantized(1).state_dict().items() if k != "state_W4"}
    with pytest.raises(RuntimeError, match="belong together"):
        m.load_state_dict(half, strict=False)
    for shape in ((16, 132), (18, 130)):
        for drop in (False, True):
            with pytest.raises(RuntimeError, match="size mismatch"):
                m.load_state_dict(_quantized(1, shape=shape, drop=drop).state_dict(), strict=False)
    with pytest.raises(RuntimeError, match="size mismatch"):
        _quantized(0, drop=True).load_state_dict(nn.Linear(132, 16).state_dict(), strict=False)
    assert all(torch.equal(v, before[k]) for k, v in m.state_dict().items() if k != "bias")
    nothing = _quantized(0)
    nothing.load_state_dict({"bias": torch.zeros(16)}, strict=False)         # no weight of either kind: the buffers stay
    assert hasattr(nothing, "W_int4")


def test_casting_a_model_changes_no_weight():
    """Scales follow into a type that holds them exactly and stay what they are otherwise, NaN included; devices and everything else follow."""
    for dtype, cast in ((torch.bfloat16, "half"), (torch.bfloat16, "float"), (torch.float16, "float"), (torch.float16, "bfloat16"), (torch.float16, "double")):
        m = _quantized(0, dtype)
        m.state_W4[0, 0] = float("nan")
        want = m.state_W4.float()
        getattr(nn.Sequential(m), cast)()
        assert m.state_W4.dtype == (torch.float16 if cast == "half" else dtype) and torch.equal(m.state_W4.float().nan_to_num(), want.nan_to_num())
        assert bool(m.state_W4[0, 0].isnan()) and m.W_int4.dtype == torch.uint8 and m.weight.dtype != dtype
    for s in (1e6, 1e-7):                                  # what fp16 does not hold
        m = _quantized(0)
        m.state_W4[3, 1] = s
        want = m.state_W4.clone()
        assert torch.equal(m.half().state_W4, want)
    exact = _quantized(0, torch.float16)
    exact.state_W4.copy_(exact.state_W4.bfloat16())
    assert exact.bfloat16().state_W4.dtype == torch.bfloat16
    assert _quantized(0).to("meta").state_W4.is_meta and _quantized(0).to("meta", torch.float16).state_W4.dtype == torch.bfloat16
