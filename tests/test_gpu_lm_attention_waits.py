"""Bounded waits of the attention of many rows: as for the row kernels, a first wait that nothing completes runs out, every warp
leaves, the error is reported once and the next call is right.  The attention of few rows has no such waits; in a call of both it
runs all the same."""
import pytest

from test_gpu_lm_attention import Batch
from test_gpu_lm_waits import stalled

pytestmark = pytest.mark.gpu


# items of whole blocks and of several, one and two column blocks, windows, both kernels in a call
@pytest.mark.parametrize("seqs,q_heads,heads,dim,window", [([(130, 130)], 4, 1, 64, 0), ([(200, 3000), (90, 500)], 8, 2, 128, 0),
                                                           ([(60, 900), (60, 60)], 8, 4, 96, 100), ([(1, 700), (300, 300), (1, 40)], 8, 2, 128, 0)])
def test_attention_tiles(seqs, q_heads, heads, dim, window):
    b = Batch(seqs, q_heads, heads, dim, 32, window=window)
    b.device_args()
    stalled(b.call, [b.out, b.lse])
