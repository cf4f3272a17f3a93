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
