"""Steps of a paged cache behind one another, each reading what the one before has just written."""
import pytest
import torch

from tests.gpu_util import DEV, assert_clean_device

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("d, page", [(128, 16), (64, 48), (256, 32)])
def test_mixed_steps_see_what_was_just_written(d, page):
    """Batches of single tokens and one part of a prompt, whose queries, lengths, tokens, tables and cache rows are written at the same addresses right before
    each call, without a wait in between: the same bits as when everything is waited for and lies elsewhere.  The part is short, so that most SMs run only
    single tokens."""
    from blockwise_int8_linear_b200 import decode_ops as o
    heads, group, B, width = 4, 2, 24, 20
    cis = o.rope_table(width * page, d, device=DEV)
    g = torch.Generator().manual_seed(1)
    cache = o.paged_kv_cache(B * width, heads, page, d, torch.bfloat16, DEV)
    for t in cache:
        t.copy_(torch.randn(t.shape, generator=g))
    room = 64
    qkv = torch.empty((room, heads * (group + 2), d), device=DEV, dtype=torch.bfloat16)
    pages, lengths, cu = (torch.empty(s, device=DEV, dtype=t) for s, t in (((B, width), torch.int32), ((B,), torch.long), ((B + 1,), torch.long)))
    steps = []
    for i in range(12):
        tokens = torch.ones(B, dtype=torch.long)
        tokens[i * 7 % B] = 9 + 2 * i                             # 18 queries of a cache head and more: the other kernel's
        steps.append([t.to(DEV) for t in (torch.randn(qkv.shape, generator=g).to(qkv.dtype), torch.randperm(B * width, generator=g).view(B, width).to(torch.int32),
                                          tokens + torch.randint(0, width * page - 64, (B,), generator=g), torch.cat((tokens.new_zeros(1), tokens.cumsum(0))))])
    want, other = [], o.PagedKVCache(*(t.clone() for t in cache))
    for x, p, n, c in steps:
        torch.cuda.synchronize()
        q = o.rope_cache_append_paged(x, cis, other, p, n, c)
        torch.cuda.synchronize()
        want.append(o.attention_paged_cache(q, other, p, n, c))
    torch.cuda.synchronize()
    got = []
    for x, p, n, c in steps:
        for to, value in ((qkv, x), (pages, p), (lengths, n), (cu, c)):
            to.copy_(value)
        q = o.rope_cache_append_paged(qkv, cis, cache, pages, lengths, cu)
        got.append(o.attention_paged_cache(q, cache, pages, lengths, cu))
        del q                                                     # the next step's queries take its place
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert all(torch.equal(a, b) for a, b in zip(cache, other))
    assert_clean_device()
