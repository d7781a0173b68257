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


def _bits(dtype, seed, shape):
    """Any 16 bits as a number of the type, and among them its largest, infinities and NaN."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randint(-32768, 32768, shape, generator=g, dtype=torch.int32).to(torch.int16).view(dtype)
    special = torch.tensor([torch.finfo(dtype).max, float("inf"), -float("inf"), float("nan")], dtype=dtype)
    return torch.where(torch.rand(shape, generator=g) < 0.5, special[torch.randint(0, 4, shape, generator=g)], x).to(DEV)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("what", ["max", "inf", "far", "bits"])
@pytest.mark.parametrize("d,rows,t", [(64, 150, 1), (128, 96, 1), (128, 96, 20), (256, 70, 3), (128, 20000, 1)])
def test_unseen_rows_may_hold_anything(d, rows, t, what, dtype):
    """Rows before the start, behind the length, and for each query those of the later ones, with the type's largest number, an infinity, 2^40
    times the visible scales (2^15 in fp16, which has no more) or any bits as scales and any codes: the same bits as without them."""
    o = _d()
    cache, k, v = _cache(1, 2, rows, d, dtype, 3)
    q = _randn((1, 4, t, d), 4, dtype)
    last, first = rows - 30, 21
    n, s = torch.tensor([last], device=DEV), torch.tensor([first], device=DEV)
    clean = o.attention_int4_cache(q, cache, n, starts=s)
    _check_attention(clean, q, k, v, [last], [first])
    fill = {"max": torch.finfo(dtype).max, "inf": float("inf"), "far": 2.0 ** 40 if dtype == BF else 2.0 ** 15}

    def spoil(rows_of):
        for codes, state in ((cache.k, cache.k_state), (cache.v, cache.v_state)):
            part = state[:, :, rows_of]
            state[:, :, rows_of] = _bits(dtype, 7, part.shape) if what == "bits" else fill[what]
            codes[:, :, rows_of] = torch.randint(0, 256, codes[:, :, rows_of].shape, dtype=torch.uint8).to(DEV)

    spoil(slice(0, first))
    spoil(slice(last, None))
    assert torch.equal(o.attention_int4_cache(q, cache, n, starts=s), clean)
    for later in range(t - 1, 0, -1):                       # the row that query `later` is the first to see
        spoil(slice(last - t + later, last - t + later + 1))
        assert torch.equal(o.attention_int4_cache(q, cache, n, starts=s)[:, :, :later], clean[:, :, :later])
    assert_clean_device()


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("at", [0, 40, 299])
def test_large_values_of_no_weight(at, dtype):
    """A row whose weight is e^-60 and whose values are 2^30 (2^15 in fp16) times the others': 8e-18 of the result, wherever it lies."""
    o = _d()
    rows, d = 300, 128
    g = torch.Generator().manual_seed(1)
    k, v = torch.randn((1, 1, rows, d), generator=g) * 0.05, torch.randn((1, 1, rows, d), generator=g)
    q = torch.ones((1, 1, 1, d))
    k[0, 0, at] = -60.0 / d ** 0.5
    v[0, 0, at] *= 2.0 ** 30 if dtype == BF else 2.0 ** 13
    kc, ks, kv = _held(k, dtype)
    vc, vs, vv = _held(v, dtype)
    q = q.to(dtype).to(DEV)
    got = o.attention_int4_cache(q, o.Int4KVCache(kc, ks, vc, vs), torch.tensor([rows], device=DEV))
    rest = [i for i in range(rows) if i != at]
    _check_attention(got, q, kv[:, :, rest], vv[:, :, rest], [rows - 1])


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_large_scores_over_many_rows(d, dtype):
    """Equal keys and values of 1 over 65536 rows, 600 sequences with scores of 60 to 3000: the result is 1.  Weights and total differ by 2^-22
    (two fp16 numbers), their sums by a step in 2^23 for every 16 of a warp's 2048 rows: 2^-15, an eighth of half a step below 1 in fp16."""
    o = _d()
    rows, b = 65536, 600
    k = torch.zeros((1, 1, 1, d))
    k[..., 0] = 1.0
    kc, ks, _ = _held(k, dtype)
    vc, vs, _ = _held(torch.ones((1, 1, 1, d)), dtype)
    cache = o.Int4KVCache(*(x.expand(-1, -1, rows, -1).contiguous().expand(b, -1, -1, -1) for x in (kc, ks, vc, vs)))
    q = torch.zeros((b, 1, 1, d), dtype=dtype, device=DEV)
    q[:, 0, 0, 0] = torch.logspace(1.78, 3.47, b).to(dtype).to(DEV)
    got = o.attention_int4_cache(q, cache, torch.tensor([rows - 5], device=DEV), scale=1.0)
    assert bool((got == 1).all()), (got.double() - 1).abs().max().item()
    assert_clean_device()


@pytest.mark.parametrize("d,rows", [(64, 600), (128, 300), (256, 100)])
def test_queries_near_the_ends_of_the_range(d, rows):
    """Queries of 1e20 let one row decide, queries of 1e-30 none; values grow by eight powers of ten along the cache."""
    o = _d()
    g = torch.Generator().manual_seed(5)
    k = torch.randn((1, 2, rows, d), generator=g)
    v = torch.randn((1, 2, rows, d), generator=g) * torch.logspace(-4, 4, rows)[:, None]
    kc, ks, kv = _held(k, BF)
    vc, vs, vv = _held(v, BF)
    q = _randn((1, 2, 1, d), 2, BF)
    q[:, 0] *= 1e20
    q[:, 1] *= 1e-30
    got = o.attention_int4_cache(q, o.Int4KVCache(kc, ks, vc, vs), torch.tensor([rows], device=DEV))
    scores = (kv[0, 0] @ q[0, 0, 0].double()) * d ** -0.5
    first, second = scores.topk(2).values.tolist()
    assert first - second > 1e-3 * first                    # far more than fp32 sums are off by
    want = vv[0, 0, scores.argmax()]
    assert bool(((got[0, 0, 0].double() - want).abs() <= want.abs() * (2.0 ** -8 + 2.0 ** -20)).all())
    _check_attention(got[:, 1:], q[:, 1:], kv[:, 1:], vv[:, 1:], [rows])


def test_rows_beyond_2_to_the_31_bytes():
    """One sequence with 2.5e9 bytes of codes: its last 300 rows are those of a short cache."""
    o = _d()
    rows, d, seen = 40_000_000, 128, 300
    short, k, v = _cache(1, 1, seen, d, BF, 12)
    big = o.int4_kv_cache(1, 1, rows, d, BF, DEV)
    for x, y in zip(big, short):
        x[:, :, rows - seen:] = y
    q = _randn((1, 4, 2, d), 13, BF)
    at = lambda n: torch.tensor([n], device=DEV)
    got = o.attention_int4_cache(q, big, at(rows), starts=at(rows - seen))
    _check_attention(got, q, k, v, [seen])
    # and with every row in sight: keys and values of 0, so that a row counts by exp(0 - its score alone)
    one = o.attention_int4_cache(q[:, :, :1], big, at(rows))
    total = torch.exp((k[0, 0] @ q[0, :, 0].double().t()) * d ** -0.5)                    # [seen, heads]
    want = torch.einsum("rh,rd->hd", total, v[0, 0]) / (total.sum(0) + rows - seen)[:, None]
    # the values that count are 300 of 4e7: sums of weights in fp32 over 128 shares, 1 part in 2^13 at the worst
    assert bool(((one[0, :, 0].double() - want).abs() <= want.abs() * 2.0 ** -8 + total.sum(0)[:, None] / rows * 2.0 ** -13).all())
