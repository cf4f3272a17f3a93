"""What the paged 4-bit cache's C entries refuse before anything reaches a GPU, beyond shapes and addresses."""
import ctypes

import pytest

from lit_llama import _native as N
from tests.test_paged_cache_host import ATTN, _struct, _with


@pytest.mark.parametrize("scale", [float("inf"), -float("inf"), 1e39, 1e-60, -0.0])
def test_scales_that_are_no_numbers_of_32_bits(scale):
    """1e39 is finite to Python and infinite to the entry; 1e-60 is 0 to it."""
    c = _struct()
    with pytest.raises(RuntimeError, match="scores times"):
        N.call("ll_kv4_attn", ctypes.addressof(c), *_with(ATTN, a8=scale))


@pytest.mark.parametrize("code", [801, 810, 820])
def test_waits_of_paged_attention_are_told_by_name(code):
    """The next look for a bounded wait that ran out names the kernels it ran out in, once."""
    N.call_ret("ll_wait_report", code)
    with pytest.raises(RuntimeError, match=f"paged attention, code {code}"):
        N.check_waits()
    N.check_waits()
