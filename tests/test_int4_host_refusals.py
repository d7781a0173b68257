"""Calls of the 4-bit operators that the C ABI refuses before it looks at a device."""
import ctypes

import pytest
import torch


@pytest.fixture(scope="module")
def L():
    if torch.cuda.is_available():
        pytest.skip("the addresses of these tests must not reach a device")
    from blockwise_int8_linear_b200 import _lib, build
    build.build()
    return _lib.lib()


def _cache(**kw):
    from blockwise_int8_linear_b200 import _lib
    return _lib.Int4Cache(*(kw.get(n, (i + 1) << 20) for i, n in enumerate(("k", "v", "k_state", "v_state"))), *([kw.get("step", 1024)] * 4),
                          *([kw.get("state_step", 64)] * 4), kw.get("max_len", 16))


def _attention(L, cache, **kw):
    one = ctypes.c_void_p(256)
    return L.bi8_attention_int4(one, 0, 8, 8, 8, ctypes.byref(cache), one, 0, None, 0, kw.get("scale", 1.0), one, kw.get("B", 2), 1, 4, 2, 128, None, 0, None)


def test_attention_refuses_a_scale_that_is_no_finite_number(L):
    assert _attention(L, _cache(), B=0) == 0
    for scale in (float("nan"), float("inf"), -float("inf"), 3e38):
        assert _attention(L, _cache(), scale=scale) == -9 and "scale" in L.bi8_last_error_string().decode()
