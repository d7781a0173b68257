"""Calls of the 4-bit operators that their Python functions refuse, one reason a test."""
import pytest
import torch

from tests.gpu_util import DEV, assert_clean_device
from tests.test_gpu_int4 import BF, HF, _d, _f, _randn, _table, _weights

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("scale", [float("nan"), float("inf"), -float("inf"), 1e39, -1e300])
def test_attention_refuses_a_scale_that_is_no_finite_number(scale):
    o = _d()
    cache = o.int4_kv_cache(1, 1, 16, 64, BF, DEV)
    with pytest.raises(ValueError, match="scale"):
        o.attention_int4_cache(_randn((1, 1, 1, 64), 1, BF), cache, torch.tensor([3], device=DEV), scale=scale)
    assert_clean_device()
