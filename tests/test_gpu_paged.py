"""The paged key/value cache on the GPU: the append bit for bit, attention against plain statements in 64 bits (``oracle/paged_oracle.py``).

Tolerance of attention, per value: half a step of the result's type; the weights' own error times sum p |v|, twice (numerator and total); and
where the weights enter the second product as one number of the type, half a step of each, times sum p |v|.  A weight's relative error: fp32
products summed over D features, at most 2^-20 of sum |q k| |scale| (D 2^-24 for D <= 256, doubled for the tensor cores' truncated
sums), in the exponent; the exponent's rounding and the exponential's, 2^-20 together with the sums over rows (thousands of rows, fp32, added
in short chains)."""
import math

import pytest
import torch

from oracle import paged_oracle as O
from tests.gpu_util import DEV, assert_clean_device

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16
HALF_STEP = {BF: 2.0 ** -8, HF: 2.0 ** -11}


def _d():
    from blockwise_int8_linear_b200 import decode_ops
    return decode_ops


def _randn(shape, seed, dtype, std=1.0):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * std).to(dtype).to(DEV)


def _long(v):
    return None if v is None else torch.tensor(v, device=DEV, dtype=torch.long)


class Batch:
    """A cache with random contents, page tables in random order with spare entries -1, and the lists that the oracle takes."""

    def __init__(self, lengths, tokens, hkv, d, page, dtype, seed, *, pad=0, packed=None, starts=None, spare_width=1, fill=None, hidden=math.nan):
        g = torch.Generator().manual_seed(seed)
        self.lengths, self.tokens, self.starts, self.page, self.dtype, self.d, self.hkv = lengths, tokens, starts, page, dtype, d, hkv
        n, b = sum(tokens), len(lengths)
        self.n = n + pad
        packed = packed if packed is not None else pad > 0 or len(set(tokens)) > 1
        self.cu = [sum(tokens[:i]) for i in range(b + 1)] if packed else None
        width = max(1, max(-(-max(x, 0) // page) for x in lengths)) + spare_width
        need = [-(-max(x, 0) // page) for x in lengths]
        order = torch.randperm(sum(need) + 2, generator=g).to(torch.int32)
        self.pages = torch.full((b, width), -1, dtype=torch.int32)
        at = 0
        for i, m in enumerate(need):
            self.pages[i, :m] = order[at:at + m]
            at += m
        o = _d()
        self.cache = o.paged_kv_cache(sum(need) + 2, hkv, page, d, dtype, DEV)
        for k, t in enumerate(self.cache):
            t.copy_(_randn(t.shape, seed + 1 + k, dtype) if fill is None else fill(t.shape, seed + 1 + k))
        # what nobody sees: rows behind the longest view, before the start, and pages of nobody
        if hidden is not None:
            seen = torch.zeros((sum(need) + 2, page), dtype=torch.bool)
            for i, x in enumerate(lengths):
                for r in range(max(0, starts[i]) if starts else 0, x):
                    seen[self.pages[i, r // page], r % page] = True
            for t in self.cache:
                t.masked_fill_(~seen.to(DEV)[:, None, :, None], hidden)

    def args(self):
        return self.pages.to(DEV), _long(self.lengths), _long(self.cu)

    def attend(self, q, **kw):
        return _d().attention_paged_cache(q, self.cache, *self.args(), starts=_long(self.starts), **kw)

    def check(self, q, got, scale=None, single=True):
        scale = q.shape[-1] ** -0.5 if scale is None else scale
        want, spread, size = O.attention(q.cpu(), self.cache.k.cpu(), self.cache.v.cpu(), self.pages, self.lengths, self.cu, self.starts, scale)
        weight = 2.0 ** -20 * size + 2.0 ** -20
        u = HALF_STEP[self.dtype]
        # fp16 has steps of 2^-24 at its lower end: a result's half step, and a weight's below 2^-14 of a total of at least 2^-8
        tiny = 2.0 ** -25
        tol = u * want.abs() + (2 * weight + (u if single else u * u)) * spread + tiny * (1 + 2 ** 8 * (spread > 0))
        assert got.dtype == q.dtype and got.shape == q.shape
        err = (got.cpu().double() - want).abs()
        assert (err <= tol).all(), f"{(err / tol).max().item()} of the tolerance at {(err / tol).argmax().item()}"
        assert_clean_device()


# ---- attention ----------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("hq, hkv", [(4, 4), (8, 2), (3, 1), (32, 1)])
@pytest.mark.parametrize("page", [16, 48])
def test_single_tokens(hq, hkv, d, page, dtype):
    b = Batch([1, 16, 17, 100, 333, 0, 47, 48, 49], [1] * 9, hkv, d, page, dtype, 1)
    q = _randn((9, hq, d), 2, dtype)
    b.check(q, b.attend(q))


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("hq, hkv", [(2, 2), (8, 2), (5, 1), (7, 1)])
@pytest.mark.parametrize("page", [16, 32, 64, 80, 128, 256])
def test_parts_of_prompts(hq, hkv, d, page, dtype):
    """Parts of 1 to 70 tokens, some with rows before them and some from the first one on, unused tokens behind."""
    b = Batch([70, 1, 200, 129, 40, 33], [70, 1, 37, 1, 40, 2], hkv, d, page, dtype, 3, pad=5)
    q = _randn((b.n, hq, d), 4, dtype)
    got = b.attend(q)
    b.check(q, got)
    assert (got[-5:] == 0).all()


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("length, tokens", [(300, 300), (129, 128), (256, 256), (257, 257), (700, 65), (1100, 130), (512, 3), (385, 127), (128, 128), (127, 127)])
def test_long_parts(length, tokens, d):
    """Tiles of queries and of rows that end on and beside their boundaries."""
    b = Batch([length, length - 1], [tokens, tokens], 1, d, 64, BF, 5)
    q = _randn((b.n, 2, d), 6, BF)
    b.check(q, b.attend(q))


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_long_caches_in_shares(d, dtype):
    """Few queries over many rows: joined within a cluster and through a workspace, sequences of very different lengths."""
    for lengths, tokens in (([3001], [1]), ([20000], [1]), ([9000, 5, 1], [1, 1, 1]), ([6000], [40]), ([5000, 17], [9, 9]), ([4000, 300, 2], [1, 30, 1])):
        b = Batch(lengths, tokens, 1, d, 32, dtype, 7)
        q = _randn((b.n, 4, d), 8, dtype)
        b.check(q, b.attend(q))


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("tokens", [[1, 1, 1, 1], [3, 1, 40, 2]])
def test_starts(d, tokens):
    """Starts on and beside boundaries, behind some of the new tokens and behind all: rows before them are not seen."""
    lengths = [200, 90, 177, 64]
    for starts in ([0, 0, 0, 0], [1, 16, 17, 63], [199, 89, 150, 64], [200, 500, 2 ** 40, -3], [128, 64, 140, 48]):
        b = Batch(lengths, tokens, 2, d, 16, BF, 9, starts=starts)
        q = _randn((b.n, 4, d), 10, BF)
        b.check(q, b.attend(q))


def test_no_tokens_and_more_tokens_than_rows():
    """Sequences without new tokens; ones whose first queries see nothing; lengths beyond the table, and below zero."""
    b = Batch([50, 30, 3, 0], [0, 7, 9, 2], 1, 64, 16, BF, 11, packed=True)
    q = _randn((b.n, 2, 64), 12, BF)
    got = b.attend(q)
    b.check(q, got)
    assert (got[7:13] == 0).all() and (got[13:16] != 0).any() and (got[16:] == 0).all()
    b = Batch([32, 48], [1, 1], 1, 64, 16, BF, 13, spare_width=0)
    q = _randn((2, 2, 64), 14, BF)
    b.lengths = [1000, -5]
    b.pages[0, 2] = b.pages[1, 0]
    got = b.attend(q)
    b.check(q, got)
    assert (got[1] == 0).all()


@pytest.mark.parametrize("tokens", [1, 3, 60])
def test_page_numbers_of_no_page_read_as_zeros(tokens):
    b = Batch([100, 100], [tokens] * 2, 1, 128, 16, BF, 15)
    b.pages[0, 2], b.pages[1, 0], b.pages[1, 5] = -7, b.cache.k.shape[0], 2 ** 31 - 1
    q = _randn((b.n, 4, 128), 16, BF)
    b.check(q, b.attend(q))


@pytest.mark.parametrize("scale", [0.0, -0.3, 1.0, 1e-30, 0.05])
@pytest.mark.parametrize("tokens", [1, 50])
def test_scales(tokens, scale):
    b = Batch([150, 77], [tokens] * 2, 2, 64, 32, BF, 17)
    q = _randn((b.n, 4, 64), 18, BF)
    b.check(q, b.attend(q, scale=scale), scale)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("tokens", [1, 50])
def test_large_scores(tokens, dtype):
    """Scores of 2^22 and 2^94 leave one row with all the weight and give no infinities or NaN."""
    d = 64
    size = 2.0 ** 14 if dtype == HF else 2.0 ** 50
    b = Batch([150, 77], [tokens] * 2, 1, d, 32, dtype, 19, fill=lambda s, seed: _randn(s, seed, dtype, 1.0))
    b.cache.k.mul_(size / 8)
    q = _randn((b.n, 2, d), 20, dtype, 1.0) * (size / 8)
    got = b.attend(q)
    want = O.attention(q.cpu(), b.cache.k.cpu(), b.cache.v.cpu(), b.pages, b.lengths, b.cu, None, d ** -0.5)[0]
    # the best two scores of a query are apart by far more than fp32 sums are off: the result is a row of v
    assert ((got.cpu().double() - want).abs() <= 2 * HALF_STEP[dtype] * want.abs() + 2.0 ** -20).all()


@pytest.mark.parametrize("tokens", [1, 3, 200])
def test_rising_scores(tokens):
    """Every row's score is above the ones before, by little and by much: the running maximum moves at each step."""
    d = 128
    for slope in (0.01, 0.3, 5.0):
        b = Batch([500], [tokens], 1, d, 16, BF, 21)
        flat = b.cache.k.view(-1, d)
        for r in range(500):
            flat[b.pages[0, r // 16] * 16 + r % 16] = 0
            flat[b.pages[0, r // 16] * 16 + r % 16, 0] = slope * r
        q = torch.zeros((b.n, 2, d), device=DEV, dtype=BF)
        q[..., 0] = 8.0
        b.check(q, b.attend(q))


@pytest.mark.parametrize("tokens", [1, 100])
def test_infinities_and_nan_of_a_sequence_are_its_own(tokens):
    """A NaN key makes its sequence's queries NaN, an infinite value leaves nothing finite in that feature; others do not notice."""
    b = Batch([200, 200, 200], [tokens] * 3, 1, 64, 16, BF, 23)
    q = _randn((b.n, 2, 64), 24, BF)
    clean = b.attend(q)
    b.cache.k[b.pages[0, 3], 0, 5, 7] = math.nan
    b.cache.v[b.pages[2, 2], 0, 4, 9] = math.inf
    got = b.attend(q)
    assert got[:tokens].isnan().all()
    assert torch.equal(got[tokens:2 * tokens], clean[tokens:2 * tokens])
    last = got[2 * tokens:]
    assert not last[..., 9].isfinite().any()
    others = [i for i in range(64) if i != 9]
    assert torch.equal(last[..., others], clean[2 * tokens:][..., others])


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("d, tokens, length", [(64, 3, 40), (128, 2, 5), (256, 4, 1000), (64, 40, 40), (128, 300, 300), (128, 90, 4000), (256, 70, 200), (64, 16, 3000)])
def test_infinities_and_nan_of_later_tokens_reach_no_earlier_query(d, tokens, length, dtype):
    """Keys and values of some of the new tokens are infinite or NaN: queries before them notice nothing, those that see them do."""
    b = Batch([length, length], [tokens, tokens], 1, d, 16, dtype, 51)
    q = _randn((b.n, 2, d), 52, dtype)
    clean = b.attend(q)
    at = lambda seq, row: (b.pages[seq, row // 16], 0, row % 16)
    first = length - tokens
    bad = {first + tokens // 2: (3, math.inf), first + tokens - 1: (d - 1, math.nan), first + tokens // 3: (17, -math.inf)}
    for row, (feature, value) in bad.items():
        b.cache.v[at(0, row)][feature] = value
    b.cache.k[at(1, length - 1)][5] = math.nan
    got = b.attend(q)
    for i in range(tokens):
        hit = [f for row, (f, _) in bad.items() if row <= first + i]
        others = [f for f in range(d) if f not in hit]
        assert torch.equal(got[i][:, others], clean[i][:, others])
        assert not got[i][:, hit].isfinite().any()
    assert torch.equal(got[tokens:-1], clean[tokens:-1]) and got[-1].isnan().all()
    assert_clean_device()


LAYOUTS = {
    "rows before heads": lambda p, h, r, d: tuple(torch.empty((p, r, h, d), device=DEV, dtype=BF).transpose(1, 2) for _ in range(2)),
    "one tensor": lambda p, h, r, d: torch.empty((p, 2, h, r, d), device=DEV, dtype=BF).unbind(1),
    "features side by side": lambda p, h, r, d: torch.empty((p, h, r, 2 * d), device=DEV, dtype=BF).split(d, dim=-1),
    "heads first": lambda p, h, r, d: tuple(torch.empty((h, p, r, d), device=DEV, dtype=BF).transpose(0, 1) for _ in range(2)),
    "wider rows": lambda p, h, r, d: tuple(torch.empty((p, h, r, d + 8), device=DEV, dtype=BF)[..., :d] for _ in range(2)),
    "some pages": lambda p, h, r, d: tuple(torch.empty((2 * p, h + 1, r, d), device=DEV, dtype=BF)[::2, 1:] for _ in range(2)),
}


@pytest.mark.parametrize("layout", list(LAYOUTS))
def test_layouts_of_the_cache_and_strided_operands(layout):
    o = _d()
    b = Batch([90, 33, 150], [1, 33, 64], 2, 64, 48, BF, 25)
    k, v = LAYOUTS[layout](*b.cache.k.shape)
    k.copy_(b.cache.k), v.copy_(b.cache.v)
    wide = _randn((b.n, 12, 64), 26, BF)
    q = wide[:, 4:8]
    dense = b.attend(q.contiguous())
    b.cache = o.PagedKVCache(k, v)
    assert torch.equal(b.attend(q), dense)
    assert torch.equal(b.attend(q.transpose(0, 1).contiguous().transpose(0, 1)), dense)
    shifted = torch.empty(b.n * 4 * 64 + 3, device=DEV, dtype=BF)[3:].view(b.n, 4, 64).copy_(q)
    assert torch.equal(b.attend(shifted), dense)
    table = torch.full((3, 2 * b.pages.shape[1] + 3), -1, dtype=torch.int32, device=DEV)
    table[:, 1:b.pages.shape[1] + 1] = b.pages.to(DEV)
    view = table[:, 1:b.pages.shape[1] + 1]
    ends = torch.tensor([[x, 0] for x in b.lengths], device=DEV)[:, 0]
    assert torch.equal(o.attention_paged_cache(q, b.cache, view, ends, _long(b.cu)), dense)
    # append into the same layout: against a dense cache
    cis = o.rope_table(200, 32, device=DEV)
    plain = o.PagedKVCache(b.cache.k.clone(memory_format=torch.contiguous_format), b.cache.v.clone(memory_format=torch.contiguous_format))
    qa, qb = (o.rope_cache_append_paged(wide[:, :8], cis, c, view, ends, _long(b.cu), layout="half") for c in (b.cache, plain))
    assert torch.equal(qa, qb) and torch.equal(b.cache.k.nan_to_num(7), plain.k.nan_to_num(7)) and torch.equal(b.cache.v.nan_to_num(7), plain.v.nan_to_num(7))
    assert_clean_device()


@pytest.mark.parametrize("d, heads, rows", [(128, 8, 4096), (64, 12, 4096), (256, 4, 2000)])
def test_many_sequences_from_cold_memory(d, heads, rows):
    """More CTAs than SMs, each with few queries of a long sequence, behind a fill of the caches: copies come late and in any order.  The reference
    is every token by itself, which takes the other kernel, and sum p |v| comes from the same call on |v|.  Tolerance: half a step of each result, half a
    step of each weight times sum p |v|, and 2^-12 of that for both calls' weights (Batch.check: at most 2^-20 (1 + sum |q k| scale), below 2^-14
    for normal values of 256 features)."""
    o = _d()
    B, T, G, page = 32, 5, 4, 64
    w = -(-rows // page)
    cache = o.paged_kv_cache(B * w, heads, page, d, BF, DEV)
    g = torch.Generator(device=DEV).manual_seed(1)
    for t in cache:
        t.copy_(torch.randn(t.shape, device=DEV, generator=g))
    pages = torch.randperm(B * w, generator=torch.Generator().manual_seed(2)).view(B, w).to(torch.int32).to(DEV)
    fill = torch.empty(64 << 20, device=DEV, dtype=torch.int32)
    for seed in (3, 4, 5):
        q = torch.randn((B, T, heads * G, d), device=DEV, generator=g).to(BF)
        n = torch.randint(rows - 300, rows + 1, (B,), generator=torch.Generator().manual_seed(seed)).to(DEV)
        alone = lambda c: torch.stack([o.attention_paged_cache(q[:, t].contiguous(), c, pages, n - T + t + 1) for t in range(T)], 1)
        want, spread = alone(cache), alone(o.PagedKVCache(cache.k, cache.v.abs())).double()
        fill.zero_()
        got = o.attention_paged_cache(q.view(B * T, heads * G, d), cache, pages, n).view_as(want)
        u = HALF_STEP[BF]
        assert ((got.double() - want.double()).abs() <= 2 * u * want.double().abs() + (u * (1 + 4 * u) + 2.0 ** -12) * spread).all()
        assert_clean_device()


def test_pages_far_apart():
    """A cache of more than 2^32 bytes a tensor whose last pages are in use."""
    o = _d()
    cache = o.paged_kv_cache(35000, 8, 64, 128, BF, DEV)          # 2.3e9 values, 4.6 GB, each
    ids = torch.tensor([[34999, 0, 34998], [17500, 34997, 1]], dtype=torch.int32)
    small = o.paged_kv_cache(6, 8, 64, 128, BF, DEV)
    for i, p in enumerate(ids.flatten().tolist()):
        for c, s, seed in ((cache.k, small.k, 1), (cache.v, small.v, 2)):
            s[i] = _randn((8, 64, 128), 10 * i + seed, BF)
            c[p] = s[i]
    here = torch.arange(6, dtype=torch.int32, device=DEV).view(2, 3)
    n, cis = torch.tensor([190, 140], device=DEV), o.rope_table(256, 128, device=DEV)
    for tokens in (1, 100):
        qkv = _randn((2 * tokens, 32, 128), 50 + tokens, BF)
        q, r = (o.rope_cache_append_paged(qkv, cis, c, t, n) for c, t in ((cache, ids.to(DEV)), (small, here)))
        assert torch.equal(q, r)
        for a, b in zip(cache, small):
            assert torch.equal(a[ids.flatten().long().to(DEV)], b)
        assert torch.equal(o.attention_paged_cache(q, cache, ids.to(DEV), n), o.attention_paged_cache(r, small, here, n))
    assert_clean_device()


# ---- append --------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("layout", ["interleaved", "half"])
@pytest.mark.parametrize("hq, hkv, d, r", [(4, 4, 64, 64), (8, 2, 128, 128), (3, 1, 256, 64), (12, 12, 64, 16), (32, 8, 128, 96), (64, 64, 256, 256)])
def test_append(hq, hkv, d, r, layout, dtype):
    """Ragged parts, single tokens, sequences without any, unused tokens behind; every other row of the cache stays what it was."""
    o = _d()
    b = Batch([70, 1, 200, 5, 129, 40], [33, 1, 17, 0, 1, 40], hkv, d, 48, dtype, 31, pad=4)
    qkv = _randn((b.n, hq + 2 * hkv, d), 32, dtype)
    cis = o.rope_table(160, r, device=DEV)                       # the third sequence's last 40 rows have no angles
    k, v = b.cache.k.cpu().clone(), b.cache.v.cpu().clone()
    want = O.append(qkv.cpu(), cis.cpu(), k, v, b.pages, b.lengths, b.cu, layout)
    got = o.rope_cache_append_paged(qkv, cis, b.cache, *b.args(), layout=layout)
    assert torch.equal(got.cpu(), want) and (got[-4:] == 0).all()
    for a, c in ((b.cache.k, k), (b.cache.v, v)):
        assert torch.equal(a.cpu().nan_to_num(7), c.nan_to_num(7)) and torch.equal(a.cpu().isnan(), c.isnan())
    assert_clean_device()


def test_append_many_sequences():
    """More sequences than threads of a block, some without tokens, one length for all."""
    o = _d()
    tokens = [(i * 7) % 3 for i in range(700)]
    b = Batch([20] * 700, tokens, 1, 64, 16, BF, 33)
    qkv = _randn((b.n, 4, 64), 34, BF)
    cis = o.rope_table(32, 64, device=DEV)
    k, v = b.cache.k.cpu().clone(), b.cache.v.cpu().clone()
    want = O.append(qkv.cpu(), cis.cpu(), k, v, b.pages, b.lengths, b.cu, "interleaved")
    got = o.rope_cache_append_paged(qkv, cis, b.cache, b.pages.to(DEV), _long([20]), _long(b.cu))
    assert torch.equal(got.cpu(), want) and torch.equal(b.cache.k.cpu().nan_to_num(7), k.nan_to_num(7)) and torch.equal(b.cache.v.cpu().nan_to_num(7), v.nan_to_num(7))
    b.check(got, o.attention_paged_cache(got, b.cache, b.pages.to(DEV), _long([20]), _long(b.cu)))


def test_append_outside_writes_nothing():
    """Positions below zero and beyond the table, pages that are none, numbers of tokens that make no sense."""
    o = _d()
    b = Batch([40, 40, 40], [2, 2, 2], 1, 64, 16, BF, 35, hidden=0.5, spare_width=0)
    qkv = _randn((6, 4, 64), 36, BF)
    cis = o.rope_table(100, 64, device=DEV)
    before = [t.clone() for t in b.cache]
    for lengths in ([1, 0, -9], [50, 10 ** 12, -2 ** 62]):
        b.lengths = lengths
        k, v = before[0].cpu().clone(), before[1].cpu().clone()
        want = O.append(qkv.cpu(), cis.cpu(), k, v, b.pages, lengths, None, "half")
        got = o.rope_cache_append_paged(qkv, cis, b.cache, *b.args(), layout="half")
        assert torch.equal(got.cpu(), want) and torch.equal(b.cache.k.cpu(), k) and torch.equal(b.cache.v.cpu(), v)
        b.cache.k.copy_(before[0]), b.cache.v.copy_(before[1])
    b.lengths = [40, 40, 40]
    b.pages[:, 2] = torch.tensor([-1, b.cache.k.shape[0], 2 ** 31 - 1], dtype=torch.int32)
    assert (o.rope_cache_append_paged(qkv, cis, b.cache, *b.args()) == 0).all()
    assert torch.equal(b.cache.k, before[0]) and torch.equal(b.cache.v, before[1])
    # numbers of tokens that go back or beyond the tensor reach no memory outside it; what they give is not defined
    for cu in ([0, 5, 2, 6], [0, 2, 4, 100], [0, -8, 4, 6], [3, 3, 3, 3]):
        q = o.rope_cache_append_paged(qkv, cis, b.cache, b.pages.to(DEV), _long(b.lengths), _long(cu))
        o.attention_paged_cache(q, b.cache, b.pages.to(DEV), _long(b.lengths), _long(cu))
        b.cache.k.copy_(before[0]), b.cache.v.copy_(before[1])
    assert_clean_device()


# ---- together ------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype, d, hq, hkv, page", [(BF, 128, 8, 2, 16), (HF, 64, 4, 4, 48), (BF, 256, 4, 1, 64)])
def test_serving_run(dtype, d, hq, hkv, page):
    """Sequences that come, are read in parts and generate tokens side by side, step by step, against a dense statement of all of it."""
    o = _d()
    g = torch.Generator().manual_seed(40)
    cis = o.rope_table(400, d, device=DEV)
    cache = o.paged_kv_cache(64, hkv, page, d, dtype, DEV)
    for t in cache:
        t.fill_(math.nan)
    free = torch.randperm(64, generator=g).tolist()
    table = torch.full((3, 12), -1, dtype=torch.int32)
    lengths, plain = [0, 0, 0], [[], [], []]
    for tokens in ([90, 0, 5], [30, 70, 1], [1, 33, 1], [1, 1, 1], [1, 1, 1], [0, 1, 60], [1, 0, 1]):
        n = sum(tokens)
        qkv = torch.randn((n + 2, hq + 2 * hkv, d), generator=g).to(dtype)
        first = 0
        for b, m in enumerate(tokens):
            plain[b].append(O.rope_float(qkv[first:first + m], cis.cpu(), torch.arange(lengths[b], lengths[b] + m), "half"))
            plain[b][-1][:, hq + hkv:] = qkv[first:first + m, hq + hkv:]
            first += m
            lengths[b] += m
            for p in range(-(-lengths[b] // page)):
                if table[b, p] < 0:
                    table[b, p] = free.pop()
        cu = [0, tokens[0], tokens[0] + tokens[1], n]
        call = (cache, table.to(DEV), _long(lengths), _long(cu))
        q = o.rope_cache_append_paged(qkv.to(DEV), cis, *call, layout="half")
        got = o.attention_paged_cache(q, *call).cpu().double()
        for b, m in enumerate(tokens):
            x = torch.cat(plain[b]).double() if plain[b] else None
            for i in range(m):
                row = lengths[b] - m + i
                assert torch.equal(q[cu[b] + i].cpu().double(), x[row, :hq])
                for h in range(hq):
                    kk, vv = x[:row + 1, hq + h // (hq // hkv)], x[:row + 1, hq + hkv + h // (hq // hkv)]
                    s = kk @ x[row, h] * d ** -0.5
                    p = torch.softmax(s, 0)
                    size = (kk * x[row, h]).abs().sum(-1).max() * d ** -0.5
                    tol = HALF_STEP[dtype] * (p @ vv).abs() + (2 * (2.0 ** -20 * size + 2.0 ** -20) + HALF_STEP[dtype]) * (p @ vv.abs()) + 2.0 ** -16
                    assert ((got[cu[b] + i, h] - p @ vv).abs() <= tol).all()
        assert (got[n:] == 0).all()
    assert_clean_device()


def test_captured_and_replayed():
    """A captured step of a batch with room for tokens: lengths, tokens and tables change between replays; a second graph has its own scratch."""
    o = _d()
    b = Batch([60, 3000, 17], [1, 1, 1], 2, 128, 32, BF, 41, hidden=None)
    cis = o.rope_table(4000, 128, device=DEV)
    pages, lengths, cu = b.pages.to(DEV), _long(b.lengths), _long([0, 1, 2, 3])
    qkv = _randn((8, 12, 128), 42, BF)

    def step():
        q = o.rope_cache_append_paged(qkv, cis, b.cache, pages, lengths, cu)
        return q, o.attention_paged_cache(q, b.cache, pages, lengths, cu)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graphs = []
    with torch.cuda.stream(s):
        step()
        s.synchronize()
        for _ in range(2):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=s):
                graphs.append((graph, step()))
    for n, c in (([60, 3000, 17], [0, 1, 2, 3]), ([61, 2500, 25], [0, 1, 1, 8]), ([64, 7, 1], [0, 4, 7, 8]), ([32, 3001, 96], [0, 0, 3, 4])):
        lengths.copy_(_long(n)), cu.copy_(_long(c))
        want_q, want = step()
        for graph, (q, out) in graphs + graphs[::-1]:
            q.zero_(), out.zero_()
            graph.replay()
            assert torch.equal(q, want_q) and torch.equal(out, want)
        b.lengths, b.cu, b.n = n, c, 8
        b.check(want_q, want)


def test_two_streams_and_repeated_runs():
    """Two calls that go through workspaces at the same time, each as it is alone; the same call gives the same bits."""
    o = _d()
    x = [Batch([9000, 8000], [1, 1], 1, 128, 64, BF, 43), Batch([5000], [40], 2, 64, 16, HF, 44)]
    q = [_randn((t.n, 4, t.d), 45 + i, t.dtype) for i, t in enumerate(x)]
    alone = [t.attend(y) for t, y in zip(x, q)]
    args = [t.args() for t in x]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(o.attention_paged_cache(q[i], x[i].cache, *args[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(t, alone[i]) for t in got[i])
    assert_clean_device()


def test_refusals():
    o = _d()
    cache = o.paged_kv_cache(4, 2, 16, 64, BF, DEV)
    for t in cache:
        t.zero_()
    pages, n, cu = torch.zeros((2, 3), dtype=torch.int32, device=DEV), _long([5, 6]), _long([0, 1, 4])
    q, qkv, cis = _randn((4, 4, 64), 1, BF), _randn((4, 8, 64), 2, BF), o.rope_table(48, 64, device=DEV)
    P = o.PagedKVCache
    attend = lambda **kw: o.attention_paged_cache(**{**dict(q=q, cache=cache, pages=pages, lengths=n, cu_tokens=cu), **kw})
    append = lambda **kw: o.rope_cache_append_paged(**{**dict(qkv=qkv, cis=cis, cache=cache, pages=pages, lengths=n, cu_tokens=cu), **kw})
    attend(), append()
    both = [
        (dict(pages=pages.long()), "int32"), (dict(pages=pages[0]), "int32"), (dict(pages=pages.cpu()), "pages"), (dict(pages=pages[:1]), "lengths|cu_tokens"),
        (dict(lengths=n.int()), "lengths"), (dict(lengths=n[:1].expand(3)), "lengths"), (dict(lengths=n.cpu()), "lengths"),
        (dict(cu_tokens=cu[:2]), "cu_tokens"), (dict(cu_tokens=cu.int()), "cu_tokens"), (dict(cu_tokens=cu.cpu()), "cu_tokens"),
        (dict(cache=P(cache.k, cache.v[:3])), "alike"), (dict(cache=P(cache.k.half(), cache.v)), "cache"), (dict(cache=P(cache.k.cpu(), cache.v)), "cache"),
        (dict(cache=P(cache.k, cache.k)), "share memory"), (dict(cache=P(cache.k[:1].expand(4, -1, -1, -1), cache.v)), "share memory"),
        (dict(cache=P(cache.k[:, :, :8], cache.v[:, :, :8])), "16"), (dict(cache=P(cache.k[..., ::2], cache.v[..., ::2])), "dense"),
        (dict(cache=P(cache.k.flatten(), cache.v)), "4-D"),
    ]
    for bad, what in both:
        for call in (attend, append):
            with pytest.raises(ValueError, match=what):
                call(**bad)
    wide = torch.zeros((4, 2, 16, 68), device=DEV, dtype=BF)
    off = torch.zeros(4 * 2 * 16 * 64 + 4, device=DEV, dtype=BF)[4:].view(4, 2, 16, 64)
    for bad, what in [(P(wide[..., :64], cache.v), "multiples of 8"), (P(off, cache.v), "16-byte")]:
        with pytest.raises(ValueError, match=what):
            attend(cache=bad)
    for bad, what in [(dict(q=q[:, :3]), "heads"), (dict(q=q[..., :32]), "head size"), (dict(q=q[0]), "expected"), (dict(q=q.half()), "cache"), (dict(q=q.float()), "bfloat16"),
                      (dict(q=q[:3], cu_tokens=None), "cu_tokens"), (dict(starts=n.int()), "starts"), (dict(scale=math.nan), "scale"), (dict(scale=1e39), "scale")]:
        with pytest.raises(ValueError, match=what):
            attend(**bad)
    for bad, what in [(dict(qkv=qkv[:, :5]), "heads"), (dict(qkv=qkv[:, :4]), "heads"), (dict(cis=cis[:, :4]), "multiple of 16"), (dict(cis=cis.cpu()), "cis"),
                      (dict(layout="other"), "layout"), (dict(qkv=qkv[:3], cu_tokens=None), "cu_tokens")]:
        with pytest.raises(ValueError, match=what):
            append(**bad)
    with pytest.raises(AssertionError):
        attend(q=q.cpu())
    import torch.autograd.forward_ad as fwd
    floats = [(attend, dict(q=q)), (append, dict(qkv=qkv)), (append, dict(cis=torch.view_as_real(cis)))]
    for call, kw in floats + [(c, dict(cache=P(cache.k.clone(), cache.v.clone()))) for c in (attend, append)]:
        (name, x), = kw.items()
        for wants in ([P(x.k.clone().requires_grad_(True), x.v), P(x.k, x.v.clone().requires_grad_(True))] if name == "cache" else [x.clone().requires_grad_(True)]):
            with pytest.raises(RuntimeError, match="backward"):
                call(**{name: wants})
            with torch.no_grad():
                call(**{name: wants})
        with fwd.dual_level(), pytest.raises(RuntimeError, match="tangent"):
            call(**{name: P(fwd.make_dual(x.k, x.k.clone()), x.v) if name == "cache" else fwd.make_dual(x, torch.ones_like(x))})
    with pytest.raises(ValueError):
        o.paged_kv_cache(4, 2, 24, 64)
    with pytest.raises(ValueError):
        o.paged_kv_cache(4, 2, 16, 80)
    with pytest.raises(ValueError):
        o.paged_kv_cache(4, 2, 16, 64, torch.float32)
    # nothing to do
    assert attend(q=q[:0], cu_tokens=_long([0, 0, 0])).shape == (0, 4, 64)
    assert append(qkv=qkv[:0], cu_tokens=None).shape == (0, 4, 64)
    empty = o.paged_kv_cache(0, 2, 16, 64, BF, DEV)
    assert (attend(cache=empty) == 0).all() and (append(cache=empty) == 0).all() and (attend(pages=pages[:, :0]) == 0).all()
    assert_clean_device()
