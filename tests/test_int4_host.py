"""What needs no GPU of the 4-bit operators: the format's arithmetic, the entry points' argument checks, the module's structure."""
import ctypes

import numpy as np
import pytest
import torch

from oracle import int4_oracle as O

F32 = np.float32


def _codes_as_the_kernel(x, s, off=0):
    """fma(x, r, 56) + 1.5 * 2^23 in fp32 (the product of a 16-bit value and an fp32 one is exact in 64 bits), r = 7/s and `off` steps."""
    r = F32(7) / s.astype(F32)
    r = (r.view(np.int32) + off).view(F32)
    v = (x.astype(np.float64) * r.astype(np.float64) + 56.0).astype(F32)
    u = v + F32(12582912.0)
    return (u.view(np.uint32) & 15).astype(np.int64) - 8


@pytest.mark.parametrize("bits", [8, 11])
def test_quantizer_arithmetic_gives_the_definition(bits):
    """Every scale and every value below it, by significands and the six exponents in which a code is not 0: 8 significant bits (bf16)
    and 11 (fp16).  rint(7 x / s) is decided by integers: 14 x against odd multiples of s."""
    m = np.arange(1 << (bits - 1), 1 << bits, dtype=np.int64)
    for sm in m[:: 1 if bits == 8 else 7]:
        for e in range(6):
            # s = sm, x = m 2^-e: both as multiples of 2^-e
            xm = m if e else m[m <= sm]
            num, den = 7 * xm, sm << e
            q, rest = num // den, num % den
            q = q + ((2 * rest > den) | ((2 * rest == den) & (q % 2 == 1)))
            x = xm.astype(F32) * F32(2.0 ** -e)
            for off in (-1, 0, 1):                         # a reciprocal that is not the nearest one
                assert np.array_equal(_codes_as_the_kernel(x, np.full(x.shape, sm, F32), off), q)
                assert np.array_equal(_codes_as_the_kernel(-x, np.full(x.shape, sm, F32), off), -q)


def test_dequantizer_arithmetic_is_the_division():
    """fma(q, a, q b) with a = s h, b = (s h - a) + s l and 1/7 = h + l, in fp32: the fp32 number nearest to s q / 7, for every significand of a
    16-bit scale (11 bits) and every code."""
    s = np.arange(1 << 10, 1 << 11, dtype=np.float64)[:, None]
    q = np.arange(-7, 8, dtype=np.float64)[None]
    h = float(F32(1.0) / F32(7.0))
    low = float(F32(1.0 / 7.0 - h))
    f = lambda t: t.astype(F32).astype(np.float64)
    a = f(s * h)
    b = f(s * low + f(s * h - a))                         # both products are exact in 64 bits
    got = (q * a + f(q * b)).astype(F32)
    assert np.array_equal(got, (s * q).astype(F32) / F32(7.0))


def test_packing_order():
    codes = torch.tensor([[-7.0, 7.0, 0.0, 1.0, -1.0]])
    assert O.pack(codes).tolist() == [[0x1 | 0xF << 4, 0x8 | 0x9 << 4, 0x7 | 0x8 << 4]]


@pytest.fixture(scope="module")
def L():
    from blockwise_int8_linear_b200 import _lib, build
    build.build()
    return _lib.lib()


def test_entry_points_validate_before_cuda(L):
    if torch.cuda.is_available():
        pytest.skip("the addresses of this test must not reach a device")
    from blockwise_int8_linear_b200 import _lib
    vp = ctypes.c_void_p
    one = vp(256)
    err = lambda: L.bi8_last_error_string().decode()
    q = lambda **kw: L.bi8_quantize_int4(kw.get("x", one), kw.get("dt", 0), kw.get("ldx", 64), one, kw.get("ldq", 32), one, kw.get("M", 4), 64,
                                         kw.get("block", 64), None)
    assert q(dt=1) == -1 and q(block=48) == -2 and q(M=-1) == -4 and q(x=None) == -8 and q(ldx=63) == -4 and q(ldq=31) == -4
    assert q(x=vp(257)) == -3 and q(M=0) == 0
    d = lambda **kw: L.bi8_dequantize_int4(one, kw.get("ldq", 32), one, kw.get("sdt", 0), kw.get("out", one), kw.get("dt", 0), 4, 64, kw.get("block", 64), None)
    assert d(sdt=1) == -1 and d(dt=7) == -1 and d(block=16) == -2 and d(ldq=16) == -4 and d(out=None) == -8 and d(out=vp(258), dt=1) == -3
    m = lambda **kw: L.bi8_matmul_int4(kw.get("x", one), kw.get("xdt", 0), kw.get("ldx", 64), one, kw.get("ldw", 32), one, None, 0, kw.get("res", None),
                                       kw.get("ldr", 64), kw.get("C", vp(1 << 20)), kw.get("ldc", 64), kw.get("dt", 0), kw.get("M", 4), 64, 64,
                                       kw.get("block", 64), None)
    assert m(xdt=1) == -1 and m(dt=9) == -1 and m(block=256) == -2 and m(ldx=8) == -4 and m(ldw=8) == -4 and m(ldc=8) == -4 and m(x=None) == -8
    assert m(C=vp(257)) == -3 and m(M=0) == 0
    assert m(res=vp((1 << 20) + 64)) == -4 and "overlap" in err()
    cache = lambda **kw: _lib.Int4Cache(*(kw.get(n, 1 << 20) for n in ("k", "v", "k_state", "v_state")), *([kw.get("step", 1024)] * 4),
                                        *([kw.get("state_step", 64)] * 4), kw.get("max_len", 16))
    ref = ctypes.byref
    a = lambda c=None, **kw: L.bi8_rope_cache_append_int4(kw.get("qkv", one), kw.get("dt", 0), one, 16, one, 0, one, ref(c or cache()), kw.get("B", 2),
                                                          kw.get("T", 1), kw.get("Hq", 4), kw.get("Hkv", 2), kw.get("D", 128), None)
    t = lambda c=None, **kw: L.bi8_attention_int4(kw.get("q", one), kw.get("dt", 0), 8, kw.get("step", 8), 8, ref(c or cache()), one, 0, None, 0, 1.0, one,
                                                  kw.get("B", 2), kw.get("T", 1), kw.get("Hq", 4), kw.get("Hkv", 2), kw.get("D", 128), None, 0, None)
    for f in (a, t):
        assert f(dt=1) == -1 and f(D=96) == -4 and f(Hq=3) == -4 and f(B=-1) == -4 and f(B=0) == 0 and f(T=0) == 0
        assert f(cache(k=None)) == -8 and f(cache(k=(1 << 20) + 4)) == -3 and f(cache(step=4)) == -3 and f(cache(state_step=1)) == -3
        assert f(cache(k_state=(1 << 20) + 2)) == -3 and f(cache(max_len=-1)) == -4
    assert a(qkv=vp(264)) == -3 and t(q=vp(264)) == -3 and t(step=4) == -3 and t(q=None) == -8
    # a long cache and few heads: the shares of the rows meet in a workspace
    assert L.bi8_attention_int4_workspace_bytes(1, 1, 8, 1, 128, 65536) > 0
    assert t(cache(max_len=65536), B=1, Hq=8, Hkv=1) == -7 and "workspace" in err()
    assert L.bi8_attention_int4_workspace_bytes(64, 1, 32, 32, 128, 65536) == 0


def test_cpu_tensors_are_refused():
    from blockwise_int8_linear_b200 import decode_ops, int4_functions as f
    x = torch.zeros(4, 64, dtype=torch.bfloat16)
    codes, state = torch.zeros(4, 32, dtype=torch.uint8), torch.zeros(4, 1, dtype=torch.bfloat16)
    cache = decode_ops.int4_kv_cache(1, 1, 8, 64, device="cpu")
    assert cache.k.shape == (1, 1, 8, 32) and cache.v_state.shape == (1, 1, 8, 1) and int(cache.k.unique()) == 0x88
    for call in (lambda: f.quantize_block_int4(x, 64), lambda: f.dequantize_block_int4(codes, state, 64), lambda: f.int4_matmul(x, codes, state, fblock_size=64),
                 lambda: decode_ops.attention_int4_cache(x.view(1, 1, 4, 64), cache, torch.ones(1, dtype=torch.int64)),
                 lambda: decode_ops.rope_cache_append_int4(torch.zeros(1, 1, 3, 64, dtype=torch.bfloat16), torch.zeros(8, 32, dtype=torch.complex64),
                                                           torch.zeros(1, dtype=torch.int64), cache)):
        with pytest.raises(AssertionError, match="cuda"):
            call()
    with pytest.raises(ValueError, match="head size"):
        decode_ops.int4_kv_cache(1, 1, 8, 80, device="cpu")
    with pytest.raises(ValueError, match="bfloat16 or float16"):
        decode_ops.int4_kv_cache(1, 1, 8, 64, torch.float32, device="cpu")


def test_replace_linear_on_cpu_module_structure():
    import torch.nn as nn
    from blockwise_int8_linear_b200 import BlockInt4Linear, BlockInt8Linear, replace_linear_with_blockwise_int4, replace_linear_with_blockwise_int8

    m = nn.Sequential(nn.Linear(8, 16), nn.ReLU(), nn.Linear(16, 4, bias=False))
    w0 = m[0].weight.data_ptr()
    replace_linear_with_blockwise_int4(m)
    assert type(m[0]) is BlockInt4Linear and type(m[2]) is BlockInt4Linear and m[0].weight.data_ptr() == w0 and m[2].bias is None
    replace_linear_with_blockwise_int8(m)                 # what has been swapped stays
    assert type(m[0]) is BlockInt4Linear
    n = nn.Sequential(nn.Linear(8, 16))
    replace_linear_with_blockwise_int8(n)
    replace_linear_with_blockwise_int4(n)
    assert type(n[0]) is BlockInt8Linear
    with pytest.raises(RuntimeError, match="inference"):
        m[0](torch.zeros(1, 8))
