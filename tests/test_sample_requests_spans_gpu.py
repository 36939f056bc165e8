"""gq_sample_requests where many logits lie close about zero and a border among them (needs a B200):
a bin's end can then be the key that stands for -0."""
import numpy as np
import pytest

from gq import CudaBackend
from test_sample_requests_gpu import check

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def g():
    be = CudaBackend(0)
    yield be
    be.close()


def about_zero(rng, n, sign, top):
    """Half of the row zeros, half numbers below 2^-126 of one sign; its largest is `top`."""
    x = np.where(rng.random(n) < 0.5, rng.integers(1, 1 << 20, n).astype(np.uint32).view(np.float32), np.float32(0))
    x *= np.float32(sign)
    x[17], x[40] = top, -top
    return x


@pytest.mark.parametrize("v", [12000, 40001, 262144])
def test_ends_that_stand_for_minus_zero(g, v):
    """Rows whose largest has ones in its last 20 bits: cut into bins of 2^20 numbers from there on, one bin ends at
    -0 (and the numbers below it follow), or begins there."""
    rng = np.random.default_rng(v)
    tops = [np.uint32(b).view(np.float32) for b in (0x3bffffff, 0x3b8fffff, 0x3f7fffff, 0x3c000000)]
    x = np.stack([about_zero(rng, v, sign, top) for top in tops for sign in (-1, 1)] * 2)
    x[8:, 17] = 3e-40  # nothing that is much larger than the rest
    m = len(x)
    f = lambda a, dt=np.float32: np.full(m, a, dt)  # noqa: E731
    for u in (np.zeros(m), f(1 - 2.0 ** -53, np.float64), rng.random(m)):
        for k in (5, v // 3, v // 2 + 9, 2 * v // 3, v - 5):
            check(g, x, k=f(k, np.int32), u=u)
        for p in (0.2, 0.55, 0.8, 0.9999):
            check(g, x, p=f(p), u=u)
        check(g, x, k=f(2 * v // 3, np.int32), p=f(0.6), u=u)
