"""Where the 4-bit cache's append writes: views, positions across the cache's ends, offsets beyond 32 bits."""
import pytest
import torch

from oracle import int4_oracle as O
from tests.gpu_util import DEV, assert_clean_device
from tests.test_gpu_int4 import BF, HF, _d, _randn, _same, _table

pytestmark = pytest.mark.gpu


def _rows(qkv, cis, hkv, dtype, table=None):
    """Codes and scales of k and of v, [B, Hkv, T, ...], for tokens at the positions of ``cis [B, T, D/2, 2]``."""
    hq = qkv.shape[2] - 2 * hkv
    k = O.rotate(qkv[:, :, hq:hq + hkv], cis[:, :, None]).transpose(1, 2)
    v = qkv[:, :, hq + hkv:].transpose(1, 2)
    out = []
    for x in (k, v):
        c, s = O.quantize(x, 64)
        out += [O.pack(c), s.to(dtype)]
    return out


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("pos", [[-1, 14], [-2, 15], [0, 13], [-3, 16]])
def test_views_and_positions_across_the_ends(pos, d, dtype):
    """Keys and values of two sequences of a larger cache, some of whose tokens lie before its first row or behind its last: every row inside
    is what the definition gives at its own position, every other row and tensor is as it was."""
    o = _d()
    rows, t, hq, hkv = 16, 3, 4, 2
    big = o.int4_kv_cache(4, 3, rows, d, dtype, DEV)
    for x in big:
        x.copy_(_randn(x.shape, 3, dtype).abs() if x.is_floating_point() else torch.randint(0, 256, x.shape, dtype=torch.uint8).to(DEV))
    want = [x.clone() for x in big]
    cache = o.Int4KVCache(*(x[1:4:2, 1:] for x in big))
    qkv, cis = _randn((2, t, hq + 2 * hkv, d), 1, dtype), _table(rows, d)
    q = o.rope_cache_append_int4(qkv, cis, torch.tensor(pos, device=DEV), cache)
    at = torch.tensor(pos, device=DEV)[:, None] + torch.arange(t, device=DEV)
    inside = (at >= 0) & (at < rows)
    turn = torch.view_as_real(cis)[at.clamp(0, rows - 1)]
    new = _rows(qkv, turn, hkv, dtype)
    wq = O.rotate(qkv[:, :, :hq], turn[:, :, None]).transpose(1, 2) * inside[:, None, :, None]
    _same(q, wq)
    for name, x in zip(("k", "k_state", "v", "v_state"), new):
        held = want[o.Int4KVCache._fields.index(name)]
        for b in range(2):
            for i in range(t):
                if inside[b, i]:
                    held[1 + 2 * b, 1:, at[b, i]] = x[b, :, i].to(held.dtype)
    for got, held in zip(big, want):
        _same(got, held)
    assert_clean_device()


def test_offsets_beyond_32_bits():
    """33 sequences of 2^20 rows, 2.2e9 bytes of codes: what the last sequence's last rows become."""
    o = _d()
    b, rows, d = 33, 1 << 20, 128
    cache = o.int4_kv_cache(b, 1, rows, d, BF, DEV)
    qkv, cis = _randn((b, 2, 3, d), 1, BF), torch.view_as_real(_table(rows, d))
    pos = torch.arange(rows - 2 - b + 1, rows - 1, device=DEV)
    o.rope_cache_append_int4(qkv, cis, pos, cache)
    at = pos[:, None] + torch.arange(2, device=DEV)
    for got, want in zip(cache, _rows(qkv, cis[at], 1, BF)):
        _same(torch.stack([got[i, 0, at[i]] for i in range(b)]), want[:, 0])
        untouched = 0x88 if got.dtype == torch.uint8 else 0
        assert int((got != untouched).any(-1).sum()) <= 2 * b
    assert_clean_device()
