"""Attention over a paged cache where a looser test would not notice: scales at the lower end of fp32, the accuracy of few queries, single rows that count, and
values that are not finite among many new tokens.  Tolerances are those of ``test_gpu_paged.Batch.check`` unless a test says otherwise."""
import math

import pytest
import torch

from tests.gpu_util import DEV, assert_clean_device
from tests.test_gpu_paged import BF, HALF_STEP, HF, Batch, _randn

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("tokens", [1, 50])
@pytest.mark.parametrize("scale", [1e-40, -3e-41, 2e-38])
def test_scales_below_the_smallest_normal_number(scale, tokens, d):
    """Queries and keys of 2^60 bring scores of 2^-10 to 2^-4 even so.  As fp32 such a scale is off by at most 2^-150: 2^-150 times a sum |q k| of 2^127.5
    at most is below 2^-22 of a weight, a quarter of what the tolerance gives it."""
    b = Batch([150, 77], [tokens] * 2, 2, d, 32, BF, 61)
    b.cache.k.mul_(2.0 ** 60)
    q = _randn((b.n, 4, d), 66, BF) * 2.0 ** 60             # not one of the keys, whose product with itself is beyond fp32
    b.check(q, b.attend(q, scale=scale), scale)


# ---- the accuracy of few queries --------------------------------------------------------------------------------------------------
def _statement(b, q, scale):
    """Per query, in 64 bits: the result, sum p |v|, the largest sum |q k| |scale|, and sum |v| times the largest weight."""
    n, hq, d = q.shape
    want, spread, size, low = (torch.zeros((n, hq, d if i != 2 else 1), dtype=torch.float64, device=DEV) for i in range(4))
    first = 0
    for i, (length, count) in enumerate(zip(b.lengths, b.tokens)):
        at = torch.arange(max(0, length))
        k, v = (t[b.pages[i, at // b.page].long(), :, at % b.page].double() for t in (b.cache.k, b.cache.v))      # [rows, heads, D]
        seen = at.to(DEV) <= length - count + torch.arange(count, device=DEV)[:, None]
        for h in range(hq):
            kk, vv, x = k[:, h // (hq // b.hkv)], v[:, h // (hq // b.hkv)], q[first:first + count, h].double()
            p = torch.softmax((x @ kk.T * scale).masked_fill(~seen, -torch.inf), -1).nan_to_num(0.0)
            part = slice(first, first + count), h
            want[part], spread[part] = p @ vv, p @ vv.abs()
            if length > 0:
                size[part] = (x.abs() @ kk.abs().T).masked_fill(~seen, 0.0).amax(-1, keepdim=True) * abs(scale)
                low[part] = p.amax(-1, keepdim=True) * (seen.double() @ vv.abs())
        first += count
    return want, spread, size, low


def few_tolerance(want, spread, size, low, dtype):
    """Weights enter the second product as two numbers of the type: half a step of half a step (u^2) of each, times sum p |v|, in the place of
    u.  fp16 has steps of 2^-24 at its lower end: half of one for every row's weight relative to the largest, and half of one for the result."""
    u = HALF_STEP[dtype]
    weight = 2.0 ** -20 * size + 2.0 ** -20
    return u * want.abs() + (2 * weight + u * u) * spread + (2.0 ** -25 * (1 + low) if dtype == HF else 0.0)


def many_tolerance(want, spread, size, low, dtype):
    """Weights as one number of the type, as in Batch.check."""
    u = HALF_STEP[dtype]
    return u * want.abs() + (2 * (2.0 ** -20 * size + 2.0 ** -20) + u) * spread + 2.0 ** -25 * (1 + 2 ** 8)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("lengths, tokens, hq, hkv", [([1, 16, 17, 100, 333, 0, 47, 48, 49], [1] * 9, 8, 2), ([60, 200], [4, 4], 4, 1), ([3001], [1], 4, 1), ([20000], [1], 8, 1),
                                                      ([9000, 5, 1], [1, 1, 1], 4, 2), ([5000, 17], [4, 4], 4, 1), ([700], [16], 2, 2)])
def test_accuracy_of_few_queries(lengths, tokens, hq, hkv, d, dtype):
    """Up to 16 queries of a cache head keep their weights in twice the bits, alone, in clusters and through a workspace."""
    b = Batch(lengths, tokens, hkv, d, 32, dtype, 71, hidden=None)
    q = _randn((b.n, hq, d), 76, dtype)
    statement = _statement(b, q, d ** -0.5)
    err = (b.attend(q).double() - statement[0]).abs()
    assert (err <= few_tolerance(*statement, dtype)).all(), (err / few_tolerance(*statement, dtype)).max().item()
    assert_clean_device()


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("lengths, tokens", [([70, 1, 200, 129, 40], [70, 1, 4, 1, 5]), ([4000, 300, 2, 900], [1, 30, 1, 4])])
def test_accuracy_in_mixed_batches(lengths, tokens, d, dtype):
    """Each sequence by its own number of queries, whatever is beside it."""
    b = Batch(lengths, tokens, 2, d, 16, dtype, 73, hidden=None)
    q = _randn((b.n, 8, d), 78, dtype)
    statement = _statement(b, q, d ** -0.5)
    few = torch.tensor([4 * t <= 16 for t in tokens for _ in range(t)], device=DEV)[:, None, None]
    tol = torch.where(few, few_tolerance(*statement, dtype), many_tolerance(*statement, dtype))
    err = (b.attend(q).double() - statement[0]).abs()
    assert (err <= tol).all(), (err / tol).max().item()
    assert_clean_device()


# ---- every row counts ---------------------------------------------------------------------------------------------------------------
def _needles(length, spare):
    """A sequence whose rows' keys are normal vectors, and the rows at and beside every boundary of 16 rows: queries that are such a row's key, at a scale of 6, give it
    all the weight but 2^-24 or less."""
    b = Batch([length], [1], 1, 64, 16, BF, 75, spare_width=spare, hidden=None)
    at = torch.arange(length)
    k, v = (t[b.pages[0, at // 16].long(), 0, at % 16] for t in (b.cache.k, b.cache.v))
    rows = torch.tensor([r for r in range(length) if r % 16 in (0, 15) or r in (1, length - 2, length - 1)], device=DEV)
    return b, k, v, rows


def _check_needles(got, k, v, rows, seen, weights):
    """`weights`: half a step of each weight that the kernel may be off by, relative."""
    for part in range(0, len(rows), 512):
        r = rows[part:part + 512]
        score = (6.0 * (k[r].double() @ k.double().T)).masked_fill(torch.arange(len(k), device=DEV) > seen[part:part + 512, None], -torch.inf)
        p = torch.softmax(score, -1)
        assert (p[torch.arange(len(r)), r] >= 1 - 2.0 ** -24).all()
    # 2^-20: the others' weights, of values up to 8, and the weights' own error (Batch.check)
    err = (got.double() - v[rows].double()).abs()
    assert (err <= (HALF_STEP[BF] + weights) * v[rows].double().abs() + 2.0 ** -20 * (8 + 1)).all(), rows[err.argmax() // got.shape[-1]].item()
    assert_clean_device()


@pytest.mark.parametrize("length, spare", [(17, 0), (900, 0), (3001, 5), (3001, 3000), (20000, 0), (70000, 7)])
def test_no_row_is_lost_by_few_queries(length, spare):
    """Alone, in shares of a cluster, and through a workspace with few and with many shares (a wider table makes more of them): 16 rows in turn."""
    b, k, v, rows = _needles(length, spare)
    rows = torch.cat((rows, rows[:1].expand(-len(rows) % 16)))
    got = torch.cat([b.attend(k[r].view(1, 16, 64), scale=6.0)[0] for r in rows.view(-1, 16)])
    _check_needles(got, k, v, rows, torch.full_like(rows, length - 1), 0.0)


@pytest.mark.parametrize("length, tokens", [(200, 200), (900, 130), (2500, 256), (5000, 300), (20000, 20)])
def test_no_row_is_lost_by_many_queries(length, tokens):
    """The same of tokens beside one another, each with rows that it sees, in one share and in several."""
    b, k, v, rows = _needles(length, 0)
    b.lengths, b.tokens, b.n = [length], [tokens], tokens
    own = length - tokens + torch.arange(tokens, device=DEV)
    at = 0
    while at < len(rows):
        r = rows[at:at + tokens]
        r = torch.cat((r, rows[:1].expand(tokens - len(r))))
        r = torch.where(r <= own, r, own)                            # rows that a token does not see: its own instead
        got = b.attend(k[r].view(tokens, 1, 64), scale=6.0)[:, 0]
        _check_needles(got, k, v, r, own, HALF_STEP[BF])
        at += tokens


# ---- values that are not finite ---------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("tokens, length, start", [(256, 256, None), (300, 300, None), (300, 420, None), (256, 4000, None), (300, 301, 190), (300, 4000, 3850)])
def test_infinities_and_nan_among_many_new_tokens(tokens, length, start, d, dtype):
    """One query head on a cache head: a tile of 256 queries ends 256 rows behind the first that not all of them see.  Bad values lie before and behind its 128th row
    and, with a long cache, in several shares; those before a start are seen by nobody."""
    b = Batch([length, length], [tokens, tokens], 1, d, 16, dtype, 81, starts=None if start is None else [start, 0])
    q = _randn((b.n, 1, d), 86, dtype)
    clean = b.attend(q)
    first = length - tokens
    bad = {first + 5: (3, math.inf), first + 127: (7, math.nan), first + 128: (11, -math.inf), first + 200: (33, math.inf), first + 250: (34, math.nan), length - 1: (d - 1, math.inf)}
    for row, (feature, value) in bad.items():
        b.cache.v[b.pages[0, row // 16], 0, row % 16][feature] = value
    got = b.attend(q)
    for i in range(tokens):
        hit = [f for row, (f, _) in bad.items() if (start or 0) <= row <= first + i]
        others = [f for f in range(d) if f not in hit]
        assert torch.equal(got[i][:, others], clean[i][:, others]), i
        assert not got[i][:, hit].isfinite().any(), i
    assert torch.equal(got[tokens:], clean[tokens:])
    assert_clean_device()
