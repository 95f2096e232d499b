"""Attention over the paged cache where values, their scales or the logits span far more than usual, against 64 bits.

U = 2^-24 is half an f32 step relative to the value; Batch and its tolerances are those of test_gpu_lm_attention.py, and
where a test needs a tighter one it is derived beside it."""
import numpy as np
import pytest

from test_gpu_lm_attention import Batch

pytestmark = pytest.mark.gpu

TOP = 0x7E  # the byte of 448


def set_values(b, value):
    """All of the cache's values to about `value`, b.v with them."""
    s = np.float32(value / 448.0)
    b.cache.v.write(np.full(b.cache.v.numel * 4, TOP, np.uint8).view(np.float32))
    b.cache.v_scale.write(np.full(b.cache.v_scale.numel, s, np.float32))
    b.v[:] = 448.0 * float(s)


@pytest.mark.parametrize("new", [1, 33])
@pytest.mark.parametrize("value,length", [(1e35, 8192), (3e38, 40), (3e38, 9000), (1e-30, 9000)])
def test_means_of_large_and_small_values(value, length, new):
    """Sums of many large values may pass f32 where their mean does not: of few rows and of many, in one block and in parts."""
    b = Batch([(new, length)], 4, 1, 64, 64)
    set_values(b, value)
    b.check()
    b.q[:] = 0.0  # equal weights
    b.check()
