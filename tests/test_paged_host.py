"""Rotary positions and the paged cache without a device: refusals of the C ABI, the tables, the oracle against itself."""
import ctypes
import math

import pytest
import torch

from oracle import paged_oracle as O


@pytest.fixture(scope="module")
def L():
    if torch.cuda.is_available():
        pytest.skip("the addresses of these tests must not reach a device")
    from blockwise_int8_linear_b200 import _lib, build
    build.build()
    return _lib.lib()


def _cache(**kw):
    from blockwise_int8_linear_b200 import _lib
    base = dict(k=1 << 20, v=1 << 21, k_page=4096, k_head=1024, k_row=64, v_page=4096, v_head=1024, v_row=64, pages=8, heads=4, page_rows=16, head_dim=64)
    return _lib.PagedCache(*({**base, **kw}[n] for n, _ in _lib.PagedCache._fields_))


def _sequences(**kw):
    from blockwise_int8_linear_b200 import _lib
    base = dict(lengths=1 << 10, cu_tokens=0, starts=0, page_table=1 << 11, lengths_step=1, starts_step=0, table_step=4, width=4, B=2, N=4)
    return _lib.Sequences(*({**base, **kw}[n] for n, _ in _lib.Sequences._fields_))


def _attention(L, cache=None, seq=None, *, q=256, dtype=0, tok=512, head=64, scale=1.0, out=256, hq=8, ws=None):
    return L.bi8_attention_paged(q, dtype, tok, head, ctypes.byref(cache or _cache()), ctypes.byref(seq or _sequences()), scale, out, hq, ws, 0, None)


def _append(L, cache=None, seq=None, *, x=256, dtype=0, tok=1024, head=64, cis=256, rows=64, R=64, layout=0, out=256, hq=8):
    return L.bi8_rope_cache_append_paged(x, dtype, tok, head, cis, rows, R, layout, out, ctypes.byref(cache or _cache()), ctypes.byref(seq or _sequences()), hq, None)


def _codes():
    import re
    from pathlib import Path
    text = (Path(__file__).parent.parent / "include" / "bi8.h").read_text()
    return {n: int(v) for n, v in re.findall(r"#define (BI8_ERR_\w+) \((-\d+)\)", text)}


@pytest.mark.parametrize("cache, seq, code", [
    (dict(pages=-1), {}, "SHAPE"), (dict(heads=0), {}, "SHAPE"), (dict(page_rows=8), {}, "SHAPE"), (dict(page_rows=24), {}, "SHAPE"), (dict(page_rows=0), {}, "SHAPE"),
    (dict(head_dim=80), {}, "SHAPE"), (dict(heads=3), {}, "SHAPE"), (dict(k=0), {}, "NULL"), (dict(v=0), {}, "NULL"), (dict(k=1 << 20 | 8), {}, "ALIGN"),
    (dict(k_row=68), {}, "ALIGN"), (dict(v_page=-8), {}, "ALIGN"), ({}, dict(B=-1), "SHAPE"), ({}, dict(N=-1), "SHAPE"), ({}, dict(N=5), "SHAPE"), ({}, dict(B=0), "SHAPE"),
    ({}, dict(width=1 << 30), "SHAPE"), ({}, dict(lengths=0), "NULL"), ({}, dict(page_table=0), "NULL"), ({}, dict(lengths=1028), "ALIGN"),
    ({}, dict(cu_tokens=1028), "ALIGN"), ({}, dict(page_table=1026), "ALIGN"), ({}, dict(table_step=-1), "SHAPE"), ({}, dict(N=1 << 30), "LIMIT")])
def test_both_calls_refuse(L, cache, seq, code):
    want = _codes()["BI8_ERR_" + code]
    assert _attention(L, _cache(**cache), _sequences(**seq)) == want
    assert _append(L, _cache(**cache), _sequences(**seq)) == want
    assert len(L.bi8_last_error_string()) > 0


@pytest.mark.parametrize("kw, code", [(dict(dtype=1), "DTYPE"), (dict(scale=math.nan), "LIMIT"), (dict(scale=math.inf), "LIMIT"), (dict(scale=-3e38), "LIMIT"),
                                      (dict(q=0), "NULL"), (dict(out=0), "NULL"), (dict(q=264), "ALIGN"), (dict(out=264), "ALIGN"), (dict(tok=516), "ALIGN"),
                                      (dict(head=-64), "ALIGN"), (dict(hq=6), "SHAPE"), (dict(hq=1 << 20), "SHAPE")])
def test_attention_refuses(L, kw, code):
    assert _attention(L, **kw) == _codes()["BI8_ERR_" + code]


@pytest.mark.parametrize("kw, code", [(dict(dtype=1), "DTYPE"), (dict(layout=2), "SHAPE"), (dict(R=8), "SHAPE"), (dict(R=40), "SHAPE"), (dict(R=80), "SHAPE"),
                                      (dict(rows=-1), "SHAPE"), (dict(x=0), "NULL"), (dict(cis=0), "NULL"), (dict(out=0), "NULL"), (dict(x=264), "ALIGN"),
                                      (dict(cis=264), "ALIGN"), (dict(tok=1020), "ALIGN")])
def test_append_refuses(L, kw, code):
    assert _append(L, **kw) == _codes()["BI8_ERR_" + code]


def test_nothing_to_do_reaches_no_device(L):
    for seq in (dict(N=0), dict(N=0, B=0)):
        assert _attention(L, seq=_sequences(**seq)) == 0 and _append(L, seq=_sequences(**seq)) == 0
    assert _attention(L, hq=0) == 0


def test_attention_wants_its_workspace(L):
    """A call of few queries over a long table goes through one; its size does not depend on a device's presence."""
    n = L.bi8_attention_paged_workspace_bytes(1, 1, 8, 4, 64, 1 << 20, 0)
    assert n > 0
    seq = _sequences(B=1, N=1, width=1 << 16)
    assert _attention(L, seq=seq) == _codes()["BI8_ERR_WORKSPACE"]
    assert L.bi8_attention_paged_workspace_bytes(1, 1, 8, 4, 96, 1 << 20, 0) == 0 and L.bi8_attention_paged_workspace_bytes(2, 3, 8, 4, 64, 64, 0) == 0


@pytest.mark.parametrize("kw, code", [
    (dict(dtype=7), "DTYPE"), (dict(layout=5), "SHAPE"), (dict(R=3), "SHAPE"), (dict(R=0), "SHAPE"), (dict(R=66), "SHAPE"), (dict(D=1), "SHAPE"), (dict(B=-1), "SHAPE"),
    (dict(x_tok=-8), "SHAPE"), (dict(x=0), "NULL"), (dict(out=0), "NULL"), (dict(cis=0), "NULL"), (dict(x=257), "ALIGN"), (dict(cis=264), "ALIGN"), (dict(pos=260), "ALIGN"),
    (dict(B=0), None), (dict(T=0), None), (dict(H=0), None)])
def test_rope_refuses(L, kw, code):
    a = {**dict(x=256, dtype=0, x_batch=1024, x_tok=256, x_head=64, cis=256, rows=8, R=64, pos=256, pos_batch=0, pos_tok=1, out=256, B=2, T=4, H=4, D=64, layout=0, conj=0), **kw}
    assert L.bi8_rope(*a.values(), None) == (0 if code is None else _codes()["BI8_ERR_" + code])


def test_functions_refuse_tensors_of_the_host():
    from blockwise_int8_linear_b200 import decode_ops as o
    cis = o.rope_table(8, 64, device="cpu")
    cache = o.paged_kv_cache(4, 2, 16, 64, device="cpu")
    pages, n = torch.zeros((1, 2), dtype=torch.int32), torch.tensor([3])
    with pytest.raises(AssertionError, match="is_cuda"):
        o.rope(torch.zeros(1, 4, 2, 64), cis)
    with pytest.raises(AssertionError, match="is_cuda"):
        o.rope_cache_append_paged(torch.zeros((1, 8, 64), dtype=torch.bfloat16), cis, cache, pages, n)
    with pytest.raises(AssertionError, match="is_cuda"):
        o.attention_paged_cache(torch.zeros((1, 4, 64), dtype=torch.bfloat16), cache, pages, n)
    with pytest.raises(ValueError, match="layout"):
        o.rope(torch.zeros(1, 4, 2, 64), cis, layout="both")


def test_tables():
    from blockwise_int8_linear_b200.decode_ops import rope_table
    t = rope_table(131072, 128, device="cpu")
    assert t.shape == (131072, 64) and t.dtype == torch.complex64
    for p, j in ((131071, 0), (131071, 1), (99999, 31), (5, 63), (0, 7)):
        a = p * 10000.0 ** (-2 * j / 128)
        # fp64 angles: their own rounding is 2^-36 at most
        assert abs(t[p, j].real.item() - math.cos(a)) <= 2.0 ** -24 and abs(t[p, j].imag.item() - math.sin(a)) <= 2.0 ** -24
    part = rope_table(16, 32, factor=8.0, parts=(1024, 1.0, 4.0), device="cpu")
    plain, full = rope_table(16, 32, device="cpu"), rope_table(16, 32, factor=8.0, device="cpu")
    turns = [1024 * 10000.0 ** (-2 * j / 32) / (2 * math.pi) for j in range(16)]
    for j, n in enumerate(turns):
        if n >= 4:
            assert torch.equal(part[:, j], plain[:, j])
        elif n <= 1:
            assert torch.equal(part[:, j], full[:, j])
        else:
            assert not torch.equal(part[:, j], plain[:, j]) and not torch.equal(part[:, j], full[:, j])
    assert rope_table(0, 2, device="cpu").shape == (0, 1)
    for bad in (dict(rows=-1, features=2), dict(rows=4, features=3), dict(rows=4, features=0), dict(rows=4, features=2, base=0.0), dict(rows=4, features=2, factor=-1.0),
                dict(rows=4, features=2, factor=math.inf), dict(rows=4, features=2, magnitude=math.nan), dict(rows=4, features=2, parts=(8, 4.0, 1.0)),
                dict(rows=4, features=2, parts=(0, 1.0, 4.0))):
        with pytest.raises(ValueError):
            rope_table(bad.pop("rows"), bad.pop("features"), device="cpu", **bad)


def test_oracle_against_a_dense_attention():
    """The oracle itself: one sequence whose pages are in order is ordinary causal attention."""
    g = torch.Generator().manual_seed(1)
    q, k, v = (torch.randn(s, generator=g) for s in ((5, 4, 8), (3, 2, 16, 8), (3, 2, 16, 8)))
    got, spread, _ = O.attention(q, k, v, torch.tensor([[0, 1, 2]], dtype=torch.int32), [40], None, None, 0.5)
    kk, vv = (t.transpose(0, 1).reshape(2, 48, 8)[:, :40].repeat_interleave(2, 0).double() for t in (k, v))
    mask = torch.arange(40)[None] <= 35 + torch.arange(5)[:, None]
    want = torch.softmax((q.double().transpose(0, 1) @ kk.transpose(1, 2) * 0.5).masked_fill(~mask, -math.inf), -1) @ vv
    assert torch.allclose(got, want.transpose(0, 1), rtol=1e-12, atol=1e-12) and (spread >= got.abs() - 1e-12).all()


def test_oracle_rotations_agree():
    g = torch.Generator().manual_seed(2)
    from blockwise_int8_linear_b200.decode_ops import rope_table
    cis = rope_table(9, 8, device="cpu")
    x, at = torch.randn((4, 3, 12), generator=g), torch.tensor([0, 8, 9, -1])
    for layout in ("half", "interleaved"):
        for conj in (False, True):
            a, b = O.rope(x, cis, at, layout, conj), O.rope_float(x, cis, at, layout, conj)
            assert (a - b).abs().max() <= 2.0 ** -22 * x.abs().max() and (b[2:] == 0).all()
        back = O.rope(O.rope(x, cis, at, layout), cis, at, layout, conj=True)
        assert (back[:2] - x[:2]).abs().max() <= 2.0 ** -22 * x.abs().max()
