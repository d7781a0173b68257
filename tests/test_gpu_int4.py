"""4-bit weights and key/value caches on the GPU, against plain statements in 64 bits (``oracle/int4_oracle.py``).

Codes, scales and dequantized values are compared bit for bit.  Tolerances of the products: half a step of the output's type at the
result's magnitude, plus what fp32 sums of the absolute values may be off by (derived at each)."""
import pytest
import torch

from oracle import int4_oracle as O
from tests.gpu_util import DEV, assert_clean_device, set_config

pytestmark = pytest.mark.gpu

BF, HF, FF = torch.bfloat16, torch.float16, torch.float32


def _f():
    from blockwise_int8_linear_b200 import int4_functions
    return int4_functions


def _d():
    from blockwise_int8_linear_b200 import decode_ops
    return decode_ops


def _randn(shape, seed, dtype, std=1.0, outliers=0.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=g) * std
    if outliers:
        x = torch.where(torch.rand(shape, generator=g) < outliers, x * 30, x)
    return x.to(dtype).to(DEV)


def _same(got, want):
    """Equal bit for bit, NaN where NaN."""
    got, want = got.cpu(), want.cpu()
    assert got.dtype == want.dtype and got.shape == want.shape
    nan = torch.isnan(want) if want.is_floating_point() else torch.zeros_like(want, dtype=torch.bool)
    assert torch.equal(torch.isnan(got) if got.is_floating_point() else nan, nan)
    assert torch.equal(got[~nan], want[~nan])


# ---- quantizer and dequantizer ---------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("block", [32, 64, 128])
@pytest.mark.parametrize("shape", [(1, 1), (3, 31), (5, 64), (2, 65), (1, 4096), (37, 1001), (64, 768), (7, 2, 3, 128), (200, 130)])
def test_quantize_and_back(shape, block, dtype):
    f = _f()
    x = _randn(shape, sum(shape) + block, dtype, 0.3, outliers=0.01)
    x.view(-1)[:: 7] = 0
    codes, state = f.quantize_block_int4(x, block)
    q, s = O.quantize(x, block)
    _same(codes, O.pack(q))
    _same(state, s.to(dtype))
    for out in (BF, HF, FF):
        v = f.dequantize_block_int4(codes, state, block, features=shape[-1], dtype=out)
        _same(v, O.values(q, s, block).float().to(out))
    assert_clean_device()


@pytest.mark.parametrize("dtype", [BF, HF])
def test_quantize_special_values(dtype):
    """Ties, all-zero blocks, the smallest and the largest magnitudes, blocks with an infinity or a NaN."""
    f = _f()
    x = torch.zeros((12, 128), dtype=dtype)
    x[0, :15] = torch.arange(-7, 8) / 2.0
    x[0, 64] = 7.0                                                     # 7 x / s is x: ties at every half
    x[0, 65:79] = torch.arange(-6, 8) - 0.5
    info = torch.finfo(dtype)
    x[2], x[3, ::3], x[4, 1] = info.max, -info.max, info.tiny
    x[5, :64] = info.tiny * info.eps                                   # the smallest denormal
    x[6, 3], x[6, 70] = float("inf"), 1.0
    x[7, 127] = float("nan")
    x[8, 5], x[8, 6] = -float("inf"), float("nan")
    x[9] = -0.0
    x[10, :40] = info.tiny * torch.linspace(0, 1, 40)
    x = x.to(DEV)
    codes, state = f.quantize_block_int4(x, 64)
    q, s = O.quantize(x, 64)
    _same(codes, O.pack(q))
    _same(state, s.to(dtype))
    for out in (dtype, FF):
        _same(f.dequantize_block_int4(codes, state, 64, dtype=out), O.values(q, s, 64).float().to(out))


def test_quantize_strided_and_offset_rows():
    f = _f()
    big = _randn((40, 3, 300), 3, BF)
    for x in (big[:, 1, 5:261], big[::2, 0, 1:200], big.transpose(0, 1)[:, :, :128], big[:, :, 7:8], big[0, 0, 3:67], big[5:6, 2, 8:72]):
        codes, state = f.quantize_block_int4(x, 64)
        q, s = O.quantize(x, 64)
        _same(codes, O.pack(q))
        _same(state, s.to(BF))
        _same(f.dequantize_block_int4(codes, state, 64, features=x.shape[-1], dtype=BF), O.values(q, s, 64).float().to(BF))
    wide = torch.zeros((40, 512), dtype=torch.uint8, device=DEV)
    codes, state = f.quantize_block_int4(big[:, 0, :256], 64)
    wide[:, 3:131] = codes
    _same(f.dequantize_block_int4(wide[:, 3:131], state, 64, dtype=BF), f.dequantize_block_int4(codes, state, 64, dtype=BF))
    for shape in ((0, 64), (4, 0), (2, 0, 64)):
        codes, state = f.quantize_block_int4(torch.zeros(shape, dtype=BF, device=DEV), 64)
        assert codes.shape == shape[:-1] + (shape[-1] // 2,) and f.dequantize_block_int4(codes, state, 64).shape == shape


# ---- matrix product --------------------------------------------------------------------------------------------------------
def _weights(n, k, block, dtype, seed, std=0.02):
    q, s = O.quantize(_randn((n, k), seed, dtype, std), block)
    return O.pack(q).to(DEV), s.to(dtype).to(DEV), O.values(q, s, block)


def _check_product(got, x, w, s, block, extra=None):
    """fp32 sums: within a block up to eight matrix instructions (sums of 16 terms that may be cut off instead of rounded, 2^-22 of their
    absolute values each, taken as 2^-19 of 8 |x| s / 7), then one rounding a block; half a step of the output."""
    x = x.double().reshape(-1, x.shape[-1])
    want = x @ w.t().to(x.device)
    if extra is not None:
        want = want + extra
    size = x.abs() @ (s.double().abs().repeat_interleave(block, -1)[:, :x.shape[1]] * (8 / 7)).t()
    if extra is not None:
        size = size + extra.abs()
    tol = want.abs() * (torch.finfo(got.dtype).eps / 2) * (1 + 2 ** -10) + size * (2 ** -19 + s.shape[1] * 2 ** -24) + torch.finfo(got.dtype).tiny
    err = (got.double().reshape(want.shape) - want).abs()
    assert bool((err <= tol).all()), ((err - tol).max().item(), (err / tol).max().item())


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("block", [32, 64, 128])
@pytest.mark.parametrize("m,k,n", [(1, 64, 1), (1, 1, 5), (2, 33, 17), (1, 4096, 512), (3, 256, 16), (8, 768, 2304), (9, 1001, 777), (16, 2048, 40),
                                   (17, 640, 129), (33, 4096, 130), (64, 520, 100), (65, 300, 70), (200, 96, 48), (1, 12000, 24),
                                   (48, 9000, 65), (12, 30000, 33), (5, 11008, 3000),
                                   (3, 832, 100), (8, 7712, 601), (20, 3904, 64)])
def test_matmul(m, k, n, block, dtype):
    f = _f()
    codes, state, w = _weights(n, k, block, dtype, m + k + n)
    x = _randn((m, k), 7 * m + n, dtype, 1.0, outliers=0.01)
    for out in (dtype, FF):
        _check_product(f.int4_matmul(x, codes, state, fblock_size=block, dtype=out), x, w, state, block)
    bias, res = _randn((n,), 5, FF), _randn((m, n), 6, dtype)
    got = f.int4_matmul(x, codes, state, bias, residual=res, fblock_size=block, dtype=dtype)
    _check_product(got, x, w, state, block, bias.double() + res.double())
    assert_clean_device()


def test_matmul_shapes_strides_and_order():
    """Leading dimensions, strided x and codes, code rows on odd addresses, a residual that is not dense, the default block and type;
    the same call gives the same bits, alone, among other rows and on another stream."""
    f = _f()
    set_config(64, BF)
    codes, state, w = _weights(300, 512, 64, BF, 1)
    x = _randn((4, 5, 512), 2, BF)
    y = f.int4_matmul(x, codes, state)
    assert y.shape == (4, 5, 300) and y.dtype == BF
    _check_product(y, x, w, state, 64)
    wide = torch.randint(0, 255, (300, 300), dtype=torch.uint8, device=DEV)
    for off in (1, 2, 8):
        wide[:, off:off + 256] = codes
        assert torch.equal(f.int4_matmul(x, wide[:, off:off + 256], state), y)
    odd = torch.zeros(300 * 8 + 1, dtype=BF, device=DEV)[1:].view(300, 8).copy_(state)        # scales that begin in a word's upper half
    assert torch.equal(f.int4_matmul(x, codes, odd), y)
    xs = torch.full((4, 5, 520), float("nan"), dtype=BF, device=DEV)
    xs[..., 3:515] = x
    assert torch.equal(f.int4_matmul(xs[..., 3:515], codes, state), y)
    assert torch.equal(f.int4_matmul(x.transpose(0, 1), codes, state), y.transpose(0, 1))
    assert torch.equal(f.int4_matmul(x[2, 3], codes, state), f.int4_matmul(x[2:3, 3], codes, state)[0])
    res = torch.zeros((20, 2, 300), dtype=BF, device=DEV)
    res[:, 1] = _randn((20, 300), 4, BF)
    got = f.int4_matmul(x.view(20, 512), codes, state, residual=res[:, 1])
    _check_product(got, x, w, state, 64, res[:, 1].double())
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        again = f.int4_matmul(x, codes, state)
    st.synchronize()
    assert torch.equal(again, y)
    for shape, n in (((0, 512), 300), ((3, 512), 0)):
        assert f.int4_matmul(torch.zeros(shape, dtype=BF, device=DEV), codes[:n], state[:n]).shape == (shape[0], n)
    bias = _randn((300,), 8, BF)
    none = f.int4_matmul(torch.zeros((3, 0), dtype=BF, device=DEV), codes[:, :0], state[:, :0], bias)
    assert torch.equal(none, bias.expand(3, 300))


def test_matmul_extreme_values():
    """Rows whose magnitudes differ by many powers of two, in one row and between rows; zero rows; a row with an infinity or a NaN; a NaN
    scale.  Everything else stays right."""
    f = _f()
    codes, state, w = _weights(64, 512, 64, BF, 11, std=1.0)
    x = _randn((6, 512), 12, BF)
    x[0] *= 1e30
    x[1] *= 1e-30
    x[2, ::2] *= 2.0 ** -20
    x[3] = 0
    x[4, 7], x[5, 500] = float("inf"), float("nan")
    y = f.int4_matmul(x, codes, state, fblock_size=64, dtype=FF)
    _check_product(y[:4], x[:4], w, state, 64)
    assert bool((y[3] == 0).all()) and not bool(torch.isfinite(y[4:]).any())
    bad = state.clone()
    bad[5, 2] = float("nan")
    z = f.int4_matmul(x[:4], codes, bad, fblock_size=64, dtype=FF)
    assert bool(torch.isnan(z[:, 5]).all())
    keep = torch.arange(64, device=DEV) != 5
    assert torch.equal(z[:, keep], y[:4, keep])


# ---- cache ------------------------------------------------------------------------------------------------------------------
def _table(rows, d):
    g = torch.Generator().manual_seed(rows + d)
    ang = torch.rand((rows, d // 2), generator=g, dtype=torch.float64) * 6.28
    return torch.complex(ang.cos().float(), ang.sin().float()).to(DEV)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("b,t,hq,hkv,d,rows", [(1, 1, 1, 1, 64, 1), (3, 1, 8, 2, 128, 20), (2, 7, 6, 6, 64, 9), (2, 5, 4, 1, 256, 40), (1, 130, 2, 2, 128, 130)])
def test_append(b, t, hq, hkv, d, rows, dtype):
    o = _d()
    cache = o.int4_kv_cache(b, hkv, rows, d, dtype, DEV)
    for x in cache:
        x.view(-1)[:] = torch.arange(x.numel(), device=DEV).to(x.dtype) % 100
    old = [x.cpu().clone() for x in cache]
    qkv, cis = _randn((b, t, hq + 2 * hkv, d), 3, dtype, 2.0), _table(rows + 3, d)
    pos = torch.tensor([(5 * i) % (rows - t + 1) for i in range(b)], device=DEV)
    q = o.rope_cache_append_int4(qkv, cis, pos, cache)
    x, pairs = qkv.cpu(), torch.view_as_real(cis.cpu())
    for i in range(b):
        p = int(pos[i])
        turn = pairs[p:p + t, None]
        _same(q[i], O.rotate(x[i, :, :hq], turn).transpose(0, 1))
        k = O.rotate(x[i, :, hq:hq + hkv], turn).transpose(0, 1)
        v = x[i, :, hq + hkv:].transpose(0, 1)
        for new, codes, state in ((k, 0, 1), (v, 2, 3)):
            c, s = O.quantize(new, 64)
            old[codes][i, :, p:p + t], old[state][i, :, p:p + t] = O.pack(c), s.to(dtype)
    for got, want in zip(cache, old):                      # new rows, and every other as it was
        _same(got, want)
    assert_clean_device()


def test_append_positions_outside_and_views():
    """Positions before, across and behind the cache's end write what is inside and nothing else; float32 pairs and complex numbers are
    the same table; a cache that is a view of some sequences of a larger one; one position for all."""
    o = _d()
    big = o.int4_kv_cache(4, 3, 16, 64, BF, DEV)
    cache = o.Int4KVCache(*(x[1:4:2, 1:] for x in big))
    qkv, cis = _randn((2, 3, 6, 64), 1, BF), _table(16, 64)
    before = [x.clone() for x in big]
    for p in (-3, 16, 2 ** 40, -2 ** 40):
        q = o.rope_cache_append_int4(qkv, cis, torch.tensor([p], device=DEV), cache)
        assert bool((q == 0).all())
        assert all(torch.equal(x, y) for x, y in zip(big, before))
    q = o.rope_cache_append_int4(qkv, cis, torch.tensor([-1, 14], device=DEV), cache)
    full = o.int4_kv_cache(2, 2, 20, 64, BF, DEV)
    want = o.rope_cache_append_int4(qkv, torch.view_as_real(cis), torch.tensor(0, device=DEV), full)
    assert bool((q[0, :, 0] == 0).all()) and not bool((want[0, :, 0] == 0).any(-1).all())
    assert bool((q[1, :, 2] == 0).all())
    for i in (0, 2):                                       # values do not depend on the position
        assert torch.equal(cache[i + 1][0, :, :2][:, :, 0] if i else cache[3][0, :, :2][:, :, 0], (full[i + 1] if i else full[3])[0, :, 1:3][:, :, 0])
    assert torch.equal(cache.v[1, :, 14:16], full.v[1, :, 0:2])
    untouched = [torch.ones(4, dtype=torch.bool) for _ in range(1)][0]
    untouched[[1, 3]] = False
    assert all(torch.equal(x[untouched], y[untouched]) and torch.equal(x[:, :1], y[:, :1]) for x, y in zip(big, before))
    short = o.rope_cache_append_int4(qkv, cis[:2], torch.tensor([0], device=DEV), full)      # a table that ends before the cache
    assert bool((short[:, :, 2] == 0).all()) and not bool((short[:, :, 1] == 0).all())


# ---- attention --------------------------------------------------------------------------------------------------------------
def _cache(b, h, rows, d, dtype, seed, k_std=1.0, v_std=1.0):
    k, s1 = O.quantize(_randn((b, h, rows, d), seed, dtype, k_std).cpu(), 64)
    v, s2 = O.quantize(_randn((b, h, rows, d), seed + 1, dtype, v_std).cpu(), 64)
    cache = _d().Int4KVCache(O.pack(k).to(DEV), s1.to(dtype).to(DEV), O.pack(v).to(DEV), s2.to(dtype).to(DEV))
    return cache, O.values(k, s1, 64).to(DEV), O.values(v, s2, 64).to(DEV)


def _check_attention(got, q, k, v, lengths, starts=None, scale=None):
    """A score is off by 2^-19 of its absolute terms (8/7 s |q|, fp32 as in the matrix product), p by twice that relatively,
    the result by that times the spread of v (2 max|v|); p v in 22 bits and fp32 sums over the rows (2^-19 + rows / 16 2^-23 of max|v|).  For
    bf16 results p * scale is one fp16 number, off by half a step, 2^-11: the result by 2^-11 sum p |v|."""
    want = O.attention(q, k, v, lengths, starts, scale)
    sc = q.shape[-1] ** -0.5 if scale is None else abs(scale)
    delta = 2 ** -19 * sc * (8 / 7) * q.double().abs().sum(-1).max().item() * k.abs().max().item()
    spread = v.abs().max().item()
    tol = want.abs() * (torch.finfo(got.dtype).eps / 2) * (1 + 2 ** -10) + spread * (4 * delta + 2 ** -19 + k.shape[2] / 16 * 2 ** -23) + torch.finfo(got.dtype).tiny
    if got.dtype == BF:
        tol = tol + 2 ** -11 * O.attention(q, k, v.abs(), lengths, starts, scale)
    err = (got.double() - want).abs()
    assert got.dtype == q.dtype and got.shape == want.shape
    assert bool((err <= tol).all()), ((err - tol).max().item(), (err / tol).max().item())


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("b,t,hq,hkv,d,rows,lengths", [
    (1, 1, 1, 1, 64, 1, [1]), (2, 1, 4, 4, 128, 40, [17, 40]), (3, 1, 32, 8, 128, 300, [0, 1, 300]), (2, 1, 16, 1, 128, 1000, [999, 64]),
    (2, 1, 8, 1, 256, 200, [200, 15]), (1, 1, 20, 2, 64, 5000, [4999]), (1, 1, 8, 1, 128, 20000, [20000]), (1, 1, 4, 4, 64, 33000, [31]),
    (2, 5, 4, 2, 128, 64, [5, 3]), (1, 40, 4, 4, 64, 100, [70]), (2, 33, 6, 2, 128, 130, [130, 20]), (1, 17, 2, 1, 256, 48, [40]),
    (1, 100, 3, 3, 128, 700, [650]), (1, 9, 8, 1, 64, 9000, [8000])])
def test_attention(b, t, hq, hkv, d, rows, lengths, dtype):
    cache, k, v = _cache(b, hkv, rows, d, dtype, rows + d)
    q = _randn((b, hq, t, d), 9, dtype, 1.5)
    n = torch.tensor(lengths, device=DEV)
    got = _d().attention_int4_cache(q, cache, n)
    _check_attention(got, q, k, v, lengths)
    assert torch.equal(got, _d().attention_int4_cache(q, cache, n))
    assert_clean_device()


def test_attention_starts_scale_and_empty_rows():
    """Left-padded sequences, a start behind the end (zeros), more queries than rows, lengths beyond the cache and below zero."""
    o = _d()
    cache, k, v = _cache(6, 2, 200, 128, BF, 5)
    q = _randn((6, 4, 3, 128), 6, BF)
    lengths, starts = [200, 150, 2, 100, 250, -5], [13, 0, 0, 100, 40, 0]
    n, s = torch.tensor(lengths, device=DEV), torch.tensor(starts, device=DEV)
    got = o.attention_int4_cache(q, cache, n, starts=s, scale=0.3)
    _check_attention(got, q, k, v, lengths, starts, 0.3)
    assert bool((got[2, :, 0] == 0).all()) and bool((got[3] == 0).all()) and bool((got[5] == 0).all())
    one = o.attention_int4_cache(q, cache, torch.tensor(77, device=DEV), starts=torch.tensor([-4], device=DEV))
    _check_attention(one, q, k, v, [77] * 6)
    assert torch.equal(o.attention_int4_cache(q, cache, torch.tensor([77] * 12, device=DEV)[::2]), one)


@pytest.mark.parametrize("rows,t", [(96, 1), (96, 20), (20000, 1)])
def test_attention_ignores_what_nobody_sees(rows, t):
    """NaN scales in every row behind the length, before the start, and (for the earlier of several queries) in the later ones' rows."""
    o = _d()
    cache, k, v = _cache(1, 2, rows, 128, BF, 3)
    q = _randn((1, 4, t, 128), 4, BF)
    last, first = rows - 30, 21
    for state in (cache.k_state, cache.v_state):
        state[:, :, last:] = float("nan")
        state[:, :, :first] = float("nan")
    got = o.attention_int4_cache(q, cache, torch.tensor([last], device=DEV), starts=torch.tensor([first], device=DEV))
    _check_attention(got, q, k[:, :, :last], v[:, :, :last], [last], [first])
    if t > 1:
        cache.k_state[:, :, last - 1] = float("nan")
        cache.v_state[:, :, last - 2] = float("nan")
        bad = o.attention_int4_cache(q, cache, torch.tensor([last], device=DEV), starts=torch.tensor([first], device=DEV))
        assert torch.equal(bad[:, :, :t - 2], got[:, :, :t - 2]) and bool(torch.isnan(bad[:, :, t - 1]).all())
        assert bool(torch.isnan(bad[:, :, t - 2]).all())


def test_attention_value_ranges():
    """Keys that decide alone, value scales that grow by many powers of two along the cache, tiny values, and large ones."""
    o = _d()
    for ks, vs in ((40.0, 1.0), (1.0, 1e-6), (1e-3, 3e4), (0.0, 1.0), (1.0, 0.0)):
        cache, k, v = _cache(2, 2, 300, 128, BF, 8, ks, vs)
        q = _randn((2, 8, 1, 128), 9, BF)
        _check_attention(o.attention_int4_cache(q, cache, torch.tensor([300, 123], device=DEV)), q, k, v, [300, 123])
    g = torch.randn((1, 2, 600, 64)) * torch.logspace(-4, 4, 600)[:, None]
    vq, s = O.quantize(g.to(BF), 64)
    cache, k, _ = _cache(1, 2, 600, 64, BF, 8)
    cache = cache._replace(v=O.pack(vq).to(DEV), v_state=s.to(BF).to(DEV))
    q = _randn((1, 2, 1, 64), 2, BF, 1e20)
    q[:, 1] = 1e-30
    _check_attention(o.attention_int4_cache(q[:, 1:], o.Int4KVCache(*(x[:, 1:] for x in cache)), torch.tensor([600], device=DEV)),
                     q[:, 1:], k[:, 1:], O.values(vq, s, 64).to(DEV)[:, 1:], [600])


def test_attention_layouts():
    """Queries as a transposed view and at an odd offset, caches that are views, one cache shared by all sequences."""
    o = _d()
    cache, k, v = _cache(3, 4, 150, 128, HF, 21)
    q = _randn((3, 8, 2, 128), 22, HF)
    n = torch.tensor([150, 60, 2], device=DEV)
    want = o.attention_int4_cache(q, cache, n)
    assert torch.equal(o.attention_int4_cache(q.transpose(1, 2).contiguous().transpose(1, 2), cache, n), want)
    off = torch.zeros(q.numel() + 1, dtype=HF, device=DEV)[1:].view(q.shape).copy_(q)
    assert torch.equal(o.attention_int4_cache(off, cache, n), want)
    part = o.Int4KVCache(*(x[::2, 1:3, :100] for x in cache))
    _check_attention(o.attention_int4_cache(q[::2, 2:6], part, n[::2] - 55 * (n[::2] > 100)), q[::2, 2:6], k[::2, 1:3, :100], v[::2, 1:3, :100], [95, 2])
    shared = o.Int4KVCache(*(x[1:2].expand(3, -1, -1, -1) for x in cache))
    _check_attention(o.attention_int4_cache(q, shared, n), q, k[1:2].expand(3, -1, -1, -1), v[1:2].expand(3, -1, -1, -1), n.tolist())
    with pytest.raises(ValueError, match="share memory"):
        o.rope_cache_append_int4(torch.zeros((3, 1, 16, 128), dtype=HF, device=DEV), _table(9, 128), n, shared)


# ---- together, streams, graphs, refusals ------------------------------------------------------------------------------------
def _decode_model(hidden, heads, kv, d, dtype, block):
    from blockwise_int8_linear_b200 import BlockInt4Linear
    set_config(block, dtype)
    qkv = BlockInt4Linear(hidden, (heads + 2 * kv) * d, bias=True, device=DEV, dtype=dtype).eval()
    out = BlockInt4Linear(heads * d, hidden, bias=False, device=DEV, dtype=dtype).eval()
    for m, seed in ((qkv, 1), (out, 2)):
        m.weight.data = _randn(m.weight.shape, seed, dtype, 0.05)
        m.prepare_for_eval(drop_weight=True)
    return qkv, out


def _layer(x, qkv, out, cis, pos, cache, heads, kv, d):
    o = _d()
    b, t, _ = x.shape
    q = o.rope_cache_append_int4(qkv(x).view(b, t, heads + 2 * kv, d), cis, pos, cache)
    att = o.attention_int4_cache(q, cache, pos + t)
    return out.infer(att.transpose(1, 2).reshape(b, t, heads * d), residual=x)


def test_layer_prompt_then_tokens_in_a_graph():
    """Projection, append, attention and output projection of one layer: a ragged prompt, then single tokens, eagerly and as a captured
    graph whose positions advance; every step against the same chain stated plainly from the kernels' own intermediate results."""
    o, f = _d(), _f()
    hidden, heads, kv, d, b = 512, 8, 2, 64, 3
    qkv, out = _decode_model(hidden, heads, kv, d, BF, 64)
    cis = _table(64, d)
    prompt, steps = _randn((b, 11, hidden), 3, BF), [_randn((b, 1, hidden), 10 + i, BF) for i in range(5)]

    def begin():
        cache = o.int4_kv_cache(b, kv, 48, d, BF, DEV)
        pos = torch.tensor([0, 4, 30], device=DEV)
        y = _layer(prompt, qkv, out, cis, pos, cache, heads, kv, d)
        pos += torch.tensor([11, 6, 11], device=DEV)       # the second prompt's last five tokens are padding, overwritten by what follows
        return cache, pos, y

    with torch.no_grad():
        cache, pos, first = begin()
        eager = []
        for x in steps:
            eager.append(_layer(x, qkv, out, cis, pos, cache, heads, kv, d).clone())
            kk = f.dequantize_block_int4(cache.k, cache.k_state, 64, dtype=FF)
            vv = f.dequantize_block_int4(cache.v, cache.v_state, 64, dtype=FF)
            proj = qkv(x).view(b, 1, heads + 2 * kv, d)
            turn = torch.view_as_real(cis)[pos][:, None, None]
            q = O.rotate(proj[:, :, :heads], turn).transpose(1, 2)
            att = o.attention_int4_cache(q, cache, pos + 1)
            _check_attention(att, q, kk.double(), vv.double(), (pos + 1).tolist())
            w = f.dequantize_block_int4(out.W_int4, out.state_W4, 64, dtype=FF).double()
            _check_product(eager[-1], att.transpose(1, 2).reshape(b, heads * d), w, out.state_W4, 64, x.double().view(b, hidden))
            pos += 1
        cache2, pos2, again = begin()
        assert torch.equal(first, again)
        x = torch.zeros_like(steps[0])
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            _layer(x, qkv, out, cis, torch.tensor([47], device=DEV), cache2, heads, kv, d)      # warm-up, in rows that nothing reads
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = _layer(x, qkv, out, cis, pos2, cache2, heads, kv, d)
            pos2.add_(1)
        for want, step in zip(eager, steps):
            x.copy_(step)
            graph.replay()
            assert torch.equal(y, want)
    assert torch.equal(pos, pos2)
    assert_clean_device()


def test_two_graphs_and_threads_share_nothing():
    """Attention with a workspace, captured twice and replayed on two streams at once, and from threads that share a stream."""
    import threading
    o = _d()
    cache, k, v = _cache(1, 1, 30000, 128, BF, 2)
    qs = [_randn((1, 8, 1, 128), s, BF) for s in range(2)]
    n = torch.tensor([30000], device=DEV)
    want = [o.attention_int4_cache(q, cache, n).clone() for q in qs]
    graphs, outs = [], []
    for q in qs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(o.attention_int4_cache(q, cache, n))
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in qs]
    torch.cuda.synchronize()
    for _ in range(20):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(outs, want))
    wrong = [0, 0]

    def work(i):
        for _ in range(50):
            wrong[i] += int(not torch.equal(o.attention_int4_cache(qs[i], cache, n), want[i]))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert wrong == [0, 0]


@pytest.mark.parametrize("weights,cache", [("int4", "int4"), ("int8", "int4"), ("int4", "bf16")])
def test_llama_driver_in_4_bits(weights, cache):
    """The inference driver at toy size with weights, cache or both in 4 bits: a captured decode step gives the eager step's tokens, and the
    prompt's logits those of the same model on the values that its 4-bit weights stand for (and a bf16 cache: keys and values within a
    14th of their block's largest, so the logits of two layers are compared loosely)."""
    import argparse

    from tests.test_gpu_models import _load
    L = _load("llama_infer")
    a = argparse.Namespace(layers=2, hidden=256, heads=4, head_dim=64, ffn=704, vocab=512, batch=2, prompt=24, decode=6, block=64,
                           weights=weights, cache=cache)
    r1, r2 = (L.run(a, rank=0, world=1, dev=torch.device(DEV), eager=e) for e in (False, True))
    assert r1["tokens"] == r2["tokens"] and len(r1["tokens"][0]) == a.decode and r1["cache"] == cache and r1["weights"] == weights
    model = L.Llama(a, torch.device(DEV), 0, 1)
    ids = torch.randint(0, a.vocab, (a.batch, a.prompt), generator=torch.Generator().manual_seed(4000)).to(DEV)
    got = model(ids, 0, 32).float()
    plain = L.Llama(argparse.Namespace(**{**vars(a), "cache": "bf16"}), torch.device(DEV), 0, 1)
    if weights == "int4":
        for m in plain.modules():
            if isinstance(m, L.Int8Linear):
                w = m.lin.dequantized_weight()
                m.lin.infer = lambda x, residual=None, w=w: torch.nn.functional.linear(x, w) + (0 if residual is None else residual)
    want = plain(ids, 0, 32).float()
    assert (got - want).norm() <= (0.02 if cache == "bf16" else 0.3) * want.norm()
    assert_clean_device()


def test_linear_module_and_checkpoints():
    from blockwise_int8_linear_b200 import BlockInt4Linear, replace_linear_with_blockwise_int4
    set_config(64, BF)
    net = torch.nn.Sequential(torch.nn.Linear(200, 130), torch.nn.Linear(130, 64, bias=False)).to(DEV)
    dense = [m.weight.detach().clone() for m in net]
    replace_linear_with_blockwise_int4(net).eval()
    x = _randn((3, 2, 200), 1, BF)
    y = net(x)                                              # fp32 weights are rounded to bf16; no gradient mode is needed for bf16 x
    assert y.shape == (3, 2, 64) and y.dtype == BF
    q, s = O.quantize(dense[0].to(BF), 64)
    _same(net[0].W_int4, O.pack(q))
    _same(net[0].dequantized_weight(), O.values(q, s, 64).float().to(BF))
    for m in net:
        m.prepare_for_eval(drop_weight=True)
        assert m.weight.numel() == 0
    assert torch.equal(net(x), y)
    other = torch.nn.Sequential(BlockInt4Linear(200, 130, device=DEV), BlockInt4Linear(130, 64, bias=False, device=DEV)).eval()
    other.load_state_dict(net.state_dict())
    assert torch.equal(other(x), y)
    set_config(64, HF)
    with pytest.raises(ValueError, match="one type"):
        net(x.to(HF))
    set_config(64, BF)


def test_refusals():
    f, o = _f(), _d()
    set_config(64, BF)
    codes, state, _ = _weights(32, 128, 64, BF, 1)
    x = _randn((2, 128), 1, BF)
    bad = [
        (ValueError, lambda: f.quantize_block_int4(x.float(), 64)), (ValueError, lambda: f.quantize_block_int4(x, 48)),
        (ValueError, lambda: f.quantize_block_int4(torch.tensor(1.0, dtype=BF, device=DEV), 64)),
        (ValueError, lambda: f.dequantize_block_int4(codes.to(torch.int8), state)), (ValueError, lambda: f.dequantize_block_int4(codes, state, features=126)),
        (ValueError, lambda: f.dequantize_block_int4(codes, state, 32)), (ValueError, lambda: f.dequantize_block_int4(codes, state.float())),
        (ValueError, lambda: f.int4_matmul(x.float(), codes, state)), (ValueError, lambda: f.int4_matmul(x[:, :64], codes, state)),
        (ValueError, lambda: f.int4_matmul(x, codes, state, fblock_size=128)), (ValueError, lambda: f.int4_matmul(x, codes, state.to(HF))),
        (ValueError, lambda: f.int4_matmul(x, codes, state, x[0, :31])), (ValueError, lambda: f.int4_matmul(x, codes, state, residual=x)),
        (ValueError, lambda: f.int4_matmul(x, codes.cpu(), state)), (ValueError, lambda: f.int4_matmul(x, codes, state, dtype=torch.float64)),
        (RuntimeError, lambda: f.int4_matmul(x.clone().requires_grad_(True), codes, state)),
        (RuntimeError, lambda: f.quantize_block_int4(x.clone().requires_grad_(True))),
    ]
    cache = o.int4_kv_cache(2, 2, 16, 64, BF, DEV)
    q, n = _randn((2, 4, 1, 64), 1, BF), torch.tensor([3], device=DEV)
    qkv, cis = _randn((2, 1, 8, 64), 1, BF), _table(16, 64)
    a = lambda q=q, cache=cache, n=n, **kw: o.attention_int4_cache(q, cache, n, **kw)
    p = lambda qkv=qkv, cis=cis, n=n, cache=cache: o.rope_cache_append_int4(qkv, cis, n, cache)
    t = lambda i, fn: o.Int4KVCache(*(fn(x) if j == i else x for j, x in enumerate(cache)))
    for call in (a, p):
        bad += [(ValueError, lambda call=call: call(n=n.int())), (ValueError, lambda call=call: call(n=torch.tensor([1, 2, 3], device=DEV))),
                (ValueError, lambda call=call: call(n=n.cpu())), (ValueError, lambda call=call: call(cache=t(0, lambda x: x[:1]))),
                (ValueError, lambda call=call: call(cache=t(1, lambda x: x.to(HF)))), (ValueError, lambda call=call: call(cache=t(2, lambda x: x[:, :, :8]))),
                (ValueError, lambda call=call: call(cache=t(3, lambda x: x.cpu()))), (ValueError, lambda call=call: call(cache=t(0, lambda x: x[..., :16]))),
                (ValueError, lambda call=call: call(cache=o.Int4KVCache(*(x[:, :, ::2] for x in cache))))]
    bad += [(ValueError, lambda: a(q[..., :32])), (ValueError, lambda: a(q[:, :3])), (ValueError, lambda: a(q.to(HF))), (ValueError, lambda: a(q.float())),
            (ValueError, lambda: a(starts=n.int())), (RuntimeError, lambda: a(q.clone().requires_grad_(True))), (ValueError, lambda: p(qkv[:, :, :7])),
            (ValueError, lambda: p(qkv[:, :, :4])), (ValueError, lambda: p(cis=cis[:, :16])), (ValueError, lambda: p(cis=cis.real.double()))]
    for error, call in bad:
        with pytest.raises(error):
            call()
    assert a(q[:, :, :0]).shape == (2, 4, 0, 64) and p(qkv[:, :0]).shape == (2, 4, 0, 64)
    empty = o.int4_kv_cache(2, 2, 0, 64, BF, DEV)
    assert bool((a(cache=empty) == 0).all()) and bool((p(cache=empty) == 0).all())
    assert_clean_device()
