"""Log probabilities' gradient at the ends of the f32 range, against 64 bits."""
import numpy as np
import pytest

from gpu_util import device

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def up(a):
    a = np.ascontiguousarray(a, np.float32)
    t = device().tensor((a.size,))
    t.write(a.reshape(-1))
    return t


@pytest.mark.parametrize("scale", [1.0, 1e9, 1e30])
@pytest.mark.parametrize("cols", [64, 4099])
def test_entropy_gradient_of_masked_logits(cols, scale):
    """A logit of -inf, or one so far below that its probability is zero, has no gradient, however large the
    entropy's gradient is (a loss scale multiplies it)."""
    d = device()
    g = np.random.default_rng([0x6D, cols])
    x = g.normal(0, 2, (4, cols)).astype(np.float32)
    x[0, ::3] = -np.inf
    x[1, 1:] = -np.inf
    x[2, ::2] = np.finfo(np.float32).min
    x[3, ::5] = -1e30
    ge = (scale * g.normal(0, 1, 4)).astype(np.float32)
    x64 = x.astype(np.float64)
    lse = np.log(np.exp(x64 - x64.max(1, keepdims=True)).sum(1)) + x64.max(1)
    p = np.exp(x64 - lse[:, None])
    ent = -np.where(p > 0, p * np.where(p > 0, x64 - lse[:, None], 0), 0).sum(1)
    l32, e32 = lse.astype(np.float32), ent.astype(np.float32)
    dx = up(np.full((4, cols), np.nan))
    d.token_logprobs_backward(4, cols, dx, up(x), None, up(l32), up(e32), None, up(ge))
    got = dx.read().reshape(4, cols)
    far = x64 - l32[:, None].astype(np.float64) < -110
    assert not got[far].any()
    dd = np.where(far, 0, x64 - l32[:, None].astype(np.float64))
    pp = np.where(far, 0, np.exp(dd))
    want = -ge[:, None].astype(np.float64) * pp * (dd + e32[:, None].astype(np.float64))
    mag = np.abs(ge[:, None].astype(np.float64)) * (np.abs(dd) + np.abs(e32[:, None]))
    # the exponential's argument rounds twice, |dd| each, then 2 units; the bracket's sum and two products
    assert np.all(np.abs(got - want) <= pp * mag * (2 * np.abs(dd) + 16) * U + 1e-37 * (1 + mag))
