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


def test_append_refuses_a_cache_whose_parts_share_memory():
    """Sequences that share heads, equal steps of sequences and heads, keys that are the values, parts that overlap by one row; and what lies
    between one another without sharing is written as any cache."""
    o = _d()
    b, h, rows, d, t = 2, 3, 16, 64, 2
    qkv, cis, n = _randn((b, t, 4 * h, d), 1, BF), _table(rows, d), torch.tensor([5, 9], device=DEV)
    qkv = torch.cat([qkv[:, :, :h], qkv[:, :, :2 * h]], 2)
    plain = o.int4_kv_cache(b, h, rows, d, BF, DEV)
    want = o.rope_cache_append_int4(qkv, cis, n, plain)
    room = torch.full((1 << 16,), 0x88, dtype=torch.uint8, device=DEV)
    state = torch.zeros(1 << 14, dtype=BF, device=DEV)
    part, scales = rows * d // 2, rows

    def cache(k_at, v_at, batch, head, ks_at=0, vs_at=4096, s_batch=h * rows, s_head=rows):
        codes = lambda at: room.as_strided((b, h, rows, d // 2), (batch, head, d // 2, 1), at)
        sc = lambda at: state.as_strided((b, h, rows, 1), (s_batch, s_head, 1, 1), at)
        return o.Int4KVCache(codes(k_at), sc(ks_at), codes(v_at), sc(vs_at))

    far = 1 << 15
    for bad in (cache(0, far, 0, part), cache(0, far, part, part), cache(0, far, 2 * part, part), cache(0, 0, h * part, part), cache(0, part, h * part, part),
                cache(0, part - d // 2, 2 * h * part, 2 * part), cache(0, far, h * part, part - d // 2), cache(0, far, h * part, part, 0, 0),
                cache(0, far, h * part, part, s_batch=rows), cache(0, far, h * part, part, 0, rows - 1, 2 * h * rows, 2 * rows), plain._replace(v=plain.k)):
        before = room.clone(), state.clone()
        with pytest.raises(ValueError, match="share memory"):
            o.rope_cache_append_int4(qkv, cis, n, bad)
        assert torch.equal(room, before[0]) and torch.equal(state, before[1])
    # heads outside, keys and values in turn, steps of 2 and 3 parts that interlock
    for good in (cache(0, far, part, 2 * part, s_batch=rows, s_head=2 * rows), cache(0, part, 2 * h * part, 2 * part, 0, rows, 2 * h * rows, 2 * rows),
                 cache(0, far, 3 * part, 2 * part)):
        for x, y in zip(good, plain):
            x.fill_(0x88 if x.dtype == torch.uint8 else 0)
        q = o.rope_cache_append_int4(qkv, cis, n, good)
        assert torch.equal(q, want) and all(torch.equal(x, y) for x, y in zip(good, plain))
    assert_clean_device()
