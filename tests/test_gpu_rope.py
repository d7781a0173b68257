"""Rotary positions on the GPU, forward and backward, against the oracle bit for bit and in 64 bits."""
import pytest
import torch

from oracle import paged_oracle as O
from tests.gpu_util import DEV, assert_clean_device

pytestmark = pytest.mark.gpu

BF, HF, FF = torch.bfloat16, torch.float16, torch.float32
HALF_STEP = {BF: 2.0 ** -8, HF: 2.0 ** -11, FF: 2.0 ** -24}      # a rounding's error, relative to the value


def _d():
    from blockwise_int8_linear_b200 import decode_ops
    return decode_ops


def _randn(shape, seed, dtype):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype).to(DEV)


def _same(got, want):
    assert got.dtype == want.dtype and got.shape == want.shape
    assert torch.equal(got.cpu(), want.cpu())


SHAPES = [(1, 1, 1, 2, 2), (2, 3, 1, 6, 2), (1, 5, 3, 7, 4), (2, 7, 5, 64, 64), (3, 33, 12, 64, 32), (1, 1, 40, 128, 128), (2, 9, 9, 96, 24), (1, 130, 4, 256, 64),
          (2, 3, 131, 8, 8), (1, 4, 3, 100, 20), (4, 2, 2, 48, 16), (1, 2, 1, 1030, 1028)]


@pytest.mark.parametrize("dtype", [BF, HF, FF])
@pytest.mark.parametrize("layout", ["interleaved", "half"])
@pytest.mark.parametrize("shape", SHAPES)
def test_rope_and_its_gradient(shape, layout, dtype):
    B, T, H, D, R = shape
    o = _d()
    cis = o.rope_table(T + 50, R, device=DEV)
    x = _randn((B, T, H, D), sum(shape), dtype).requires_grad_(True)
    g = _randn((B, T, H, D), sum(shape) + 1, dtype)
    for positions in (None, torch.arange(T, device=DEV) + 50, torch.randint(0, T + 50, (B, T), generator=torch.Generator().manual_seed(3)).to(DEV)):
        y = o.rope(x, cis, positions, layout=layout)
        at = (torch.arange(T) if positions is None else positions.cpu()).expand(B, T)
        _same(y, O.rope_float(x.detach().cpu(), cis.cpu(), at, layout))
        gx, = torch.autograd.grad(y, x, g)
        _same(gx, O.rope_float(g.cpu(), cis.cpu(), at, layout, conj=True))
        # products and sums of two terms: two roundings of 2^-24 of |x c| + |y s|, at most 2^-22 of the largest value, and the type's own
        want = O.rope(x.detach().cpu(), cis.cpu(), at, layout)
        top = x.detach().abs().max().item()
        assert ((y.detach().cpu().double() - want).abs() <= HALF_STEP[dtype] * want.abs() + 2.0 ** -22 * top + 2.0 ** -25).all()
    assert_clean_device()


@pytest.mark.parametrize("layout", ["interleaved", "half"])
def test_gradient_against_differences(layout):
    """A linear function's difference quotient is exact but for roundings: multiples of 2^-10 up to 5, differences of 1 / 8."""
    o = _d()
    cis = o.rope_table(9, 8, device=DEV)
    x = (_randn((2, 9, 2, 12), 1, FF) * 1024).round().div(1024).clamp(-5, 5).requires_grad_(True)
    g = _randn((2, 9, 2, 12), 2, FF).clamp(-5, 5)
    gx, = torch.autograd.grad(o.rope(x, cis, layout=layout), x, g)
    step = torch.zeros_like(x)
    for i in range(0, x.numel(), 11):
        step.zero_().view(-1)[i] = 0.125
        with torch.no_grad():
            d = ((o.rope(x + step, cis, layout=layout).double() - o.rope(x - step, cis, layout=layout).double()) * g.double()).sum() / 0.25
        # two features, each a difference of two values that are off by 2 * 2^-24 of |x c| + |y s| <= 8, times |g| over 1/4; the gradient itself
        assert abs(d.item() - gx.view(-1)[i].item()) <= 2 * 2 * 2.0 ** -23 * 8 * 5 * 4 + 2.0 ** -23 * 8


def test_second_derivative_is_the_rotation():
    o = _d()
    cis = o.rope_table(5, 16, device=DEV)
    x, g, w = (_randn((1, 5, 2, 16), s, FF) for s in (1, 2, 3))
    x.requires_grad_(True)
    g.requires_grad_(True)
    gx, = torch.autograd.grad(o.rope(x, cis, layout="half"), x, g, create_graph=True)
    gg, = torch.autograd.grad(gx, g, w)
    _same(gg, o.rope(w, cis, layout="half"))


def test_positions_outside_the_table_are_zeros():
    o = _d()
    cis = o.rope_table(4, 16, device=DEV)
    x = _randn((1, 6, 3, 32), 1, BF).requires_grad_(True)
    at = torch.tensor([-1, 0, 3, 4, 2 ** 40, -2 ** 62], device=DEV)
    y = o.rope(x, cis, at)
    gx, = torch.autograd.grad(y, x, torch.ones_like(y))
    for t in (y, gx):
        assert (t[:, [0, 3, 4, 5]] == 0).all() and (t[:, 1:3] != 0).any()
    _same(o.rope(x.detach(), cis[:0], at), torch.zeros_like(x))


@pytest.mark.parametrize("dtype", [BF, FF])
def test_any_strides(dtype):
    """Views of a fused projection, transposed and expanded ones, rows that begin anywhere, features that are not dense, an expanded gradient."""
    o = _d()
    cis = o.rope_table(10, 32, device=DEV)
    base = _randn((2, 10, 9, 64), 1, dtype)
    off = torch.empty(2 * 10 * 9 * 64 + 1, device=DEV, dtype=dtype)[1:].view(2, 10, 9, 64).copy_(base)
    views = [base[:, :, 2:7], base.transpose(1, 2)[:, :, :10], base[:, ::2], base[:1].expand(3, -1, -1, -1), off, base[..., ::2], base[..., 1:49], base[0], base[:, :, :1],
             base.permute(3, 1, 2, 0)[:4, :, :, :].repeat(1, 1, 1, 16)]
    for x in views:
        T = x.shape[-3]
        at = torch.arange(T)
        want = O.rope_float(x.cpu(), cis.cpu(), at.expand(x.shape[:-2]), "half") if x.dim() == 4 else O.rope_float(x.cpu(), cis.cpu(), at, "half")
        _same(o.rope(x, cis, layout="half"), want)
    x = base.clone().requires_grad_(True)
    gx, = torch.autograd.grad(o.rope(x, cis).sum(), x)
    _same(gx, O.rope_float(torch.ones_like(base).cpu(), cis.cpu(), torch.arange(10).expand(2, 10), "interleaved", conj=True))
    # broadcast heads: their gradients are summed by the expansion's own backward pass
    one = base[:, :, :1].clone().requires_grad_(True)
    gx, = torch.autograd.grad(o.rope(one.expand(-1, -1, 4, -1), cis), one, base[:, :, :4])
    turned = O.rope_float(base[:, :, :4].cpu(), cis.cpu(), torch.arange(10).expand(2, 10), "interleaved", conj=True)
    assert ((gx.cpu().double() - turned.double().sum(2, keepdim=True)).abs() <= 4 * HALF_STEP[dtype] * turned.double().abs().sum(2, keepdim=True)).all()


def test_values_that_another_tensor_holds_negated():
    """The imaginary part of a conjugated tensor is a view whose memory has the other sign."""
    o = _d()
    cis = o.rope_table(6, 16, device=DEV)
    z = torch.complex(_randn((2, 6, 3, 32), 1, FF), _randn((2, 6, 3, 32), 2, FF))
    x = z.conj().imag
    assert x.is_neg()
    _same(o.rope(x, cis), o.rope(-z.imag, cis))
    q = _randn((3, 4, 64), 3, BF)
    cache = o.paged_kv_cache(2, 2, 16, 64, BF, DEV)
    with pytest.raises(ValueError, match="negated"):
        o.attention_paged_cache(q, o.PagedKVCache(torch._neg_view(cache.k), cache.v), torch.zeros((3, 1), dtype=torch.int32, device=DEV), torch.tensor([1], device=DEV))
    cache.k.copy_(_randn(cache.k.shape, 4, BF)), cache.v.copy_(_randn(cache.v.shape, 5, BF))
    args = cache, torch.zeros((3, 1), dtype=torch.int32, device=DEV), torch.tensor([9], device=DEV)
    _same(o.attention_paged_cache(torch._neg_view(q), *args), o.attention_paged_cache(-q, *args))


def test_tables_of_both_forms_and_any_place():
    o = _d()
    cis = o.rope_table(12, 64, device=DEV)
    x = _randn((2, 12, 3, 64), 1, BF)
    want = o.rope(x, cis)
    _same(o.rope(x, torch.view_as_real(cis)), want)
    shifted = torch.empty(12 * 64 + 2, device=DEV)[2:].view(12, 32, 2).copy_(torch.view_as_real(cis))
    _same(o.rope(x, shifted), want)
    _same(o.rope(x, cis.conj().clone().conj()), want)
    wide = torch.empty((12, 40), device=DEV, dtype=torch.complex64)
    wide[:, :32] = cis
    _same(o.rope(x, wide[:, :32]), want)


def test_scaled_tables():
    """The scaled table against the formula in 64 bits, pair by pair."""
    import math
    o = _d()
    t = o.rope_table(1000, 64, base=500000.0, factor=8.0, parts=(8192, 1.0, 4.0), magnitude=1.25, device=DEV).cpu()
    for j in range(32):
        w = 500000.0 ** (-2 * j / 64)
        turns = 8192 * w / (2 * math.pi)
        keep = min(1.0, max(0.0, (turns - 1.0) / 3.0))
        w = keep * w + (1 - keep) * w / 8.0
        for p in (0, 1, 999):
            # |cos| up to 1.25 in fp32; angles up to 1000 in 64 bits
            assert abs(t[p, j].real.item() - 1.25 * math.cos(p * w)) <= 2.0 ** -24 and abs(t[p, j].imag.item() - 1.25 * math.sin(p * w)) <= 2.0 ** -24
    plain, stretched = o.rope_table(64, 16, device=DEV), o.rope_table(64, 16, factor=4.0, device=DEV)
    assert torch.equal(plain[::2], o.rope_table(32, 16, device=DEV, factor=0.5))
    assert not torch.equal(plain, stretched) and torch.allclose(stretched[::4], plain[:16], rtol=0, atol=2.0 ** -23)


def test_refusals():
    o = _d()
    cis = o.rope_table(4, 16, device=DEV)
    x = _randn((1, 4, 2, 32), 1, BF)
    for bad, what in [((x[0, 0], cis), "expected"), ((x, cis[:, :0]), "pairs"), ((x[..., :8], cis), "pairs"), ((x, cis.real), "cis"), ((x, cis.to(torch.complex128)), "cis"),
                      ((x, cis.cpu()), "cis"), ((x.double(), cis), "dtype"), ((x, cis, torch.arange(4, device=DEV).int()), "positions"),
                      ((x, cis, torch.arange(3, device=DEV)), "positions"), ((x, cis, torch.zeros((2, 4), device=DEV, dtype=torch.long)), "positions"),
                      ((x[0], cis, torch.zeros((1, 4), device=DEV, dtype=torch.long)), "positions"), ((x, cis, torch.arange(4)), "positions")]:
        with pytest.raises(ValueError, match=what):
            o.rope(*bad)
    with pytest.raises(ValueError, match="layout"):
        o.rope(x, cis, layout="neox")
    with pytest.raises(AssertionError):
        o.rope(x.cpu(), cis)
    with pytest.raises(RuntimeError, match="table"):
        o.rope(x, torch.view_as_real(cis).clone().requires_grad_(True))
    import torch.autograd.forward_ad as fwd
    with fwd.dual_level(), pytest.raises(RuntimeError, match="tangent"):
        o.rope(fwd.make_dual(x, torch.ones_like(x)), cis)
    y = o.rope(x.clone().requires_grad_(True), cis, at := torch.arange(4, device=DEV))
    at.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    assert o.rope(x[:0], cis).shape == (0, 4, 2, 32) and o.rope(x[:, :0], cis).numel() == 0
    assert_clean_device()


def test_streams_and_graphs():
    """On another stream than the default one, and in a captured training step whose positions advance between replays."""
    o = _d()
    cis = o.rope_table(64, 32, device=DEV)
    x = _randn((2, 8, 3, 32), 1, BF)
    at = torch.arange(8, device=DEV)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        y = o.rope(x, cis, at)
    s.synchronize()
    _same(y, O.rope_float(x.cpu(), cis.cpu(), torch.arange(8).expand(2, 8), "interleaved"))
    leaf = x.clone().requires_grad_(True)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(s):
        torch.autograd.grad(o.rope(leaf, cis, at).float().square().sum(), leaf)
    s.synchronize()
    with torch.cuda.graph(graph, stream=s):
        y = o.rope(leaf, cis, at)
        g, = torch.autograd.grad(y, leaf, x)
        y = y.detach()
    for shift in (0, 5, 50):
        at.copy_(torch.arange(8, device=DEV) + shift)
        graph.replay()
        torch.cuda.synchronize()
        want = (torch.arange(8) + shift).expand(2, 8)
        _same(y, O.rope_float(x.cpu(), cis.cpu(), want, "interleaved"))
        _same(g, O.rope_float(x.cpu(), cis.cpu(), want, "interleaved", conj=True))
    assert_clean_device()


def test_offsets_beyond_32_bits():
    """More than 2^32 bytes and 2^31 values: the last tokens."""
    o = _d()
    cis = o.rope_table(2, 16, device=DEV)
    x = torch.zeros((70000, 2, 128, 128), device=DEV, dtype=BF)
    x[-1] = _randn((2, 128, 128), 1, BF)
    y = o.rope(x, cis, torch.tensor([0, 1], device=DEV))
    _same(y[-1:], O.rope_float(x[-1:].cpu(), cis.cpu(), torch.tensor([[0, 1]]), "interleaved"))
    assert not y[:-1].any()
