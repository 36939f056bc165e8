"""Greedy rows of gq_sample_requests (needs a B200): the first of the largest, whatever else is large in its
piece of the row, also in more places than a piece gives keys of."""
import numpy as np
import pytest

from gq import CudaBackend
from test_sample_requests_gpu import check, dev

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def g():
    be = CudaBackend(0)
    yield be
    be.close()


@pytest.mark.parametrize("v", [32003, 262144])
@pytest.mark.parametrize("m", [1, 37, 64])
def test_greedy_rows(g, m, v):
    rng = np.random.default_rng(m * 7 + v)
    zero = np.zeros(m, np.float32)
    x = rng.standard_normal((m, v)).astype(np.float32)
    rising, falling, eights, ties, some = (x.copy() for _ in range(5))
    rising[:, 1000:1100] = np.linspace(5, 9, 100, dtype=np.float32)  # the largest is the last of its neighbours
    falling[:, 1000:1100] = np.linspace(9, 5, 100, dtype=np.float32)
    at = rng.integers(0, v // 8, (m, 40)) * 8  # eight ids at a time nearly equal
    for i in range(m):
        for a in at[i]:
            eights[i, a:a + 8] = rng.uniform(3, 9) + np.arange(8) * 1e-4
    ties[:] = rng.choice([-3.25, 0.0, 7.5], (m, 1))  # a row of one number
    some[:] = np.round(some * 2) / 2  # few numbers, the largest of them anywhere
    some[:, :200] = -9.0
    some[:, 4000:9000] = 6.0
    for y in (rising, falling, eights, ties, some):
        for u in (rng.random(m), np.full(m, 1 - 2.0 ** -53)):
            check(g, y, t=zero, u=u)
            check(g, y, t=zero, k=rng.choice([0, 3, 1000], m).astype(np.int32), p=np.full(m, 0.5, np.float32), u=u)


def test_greedy_is_the_same_from_run_to_run(g):
    """64 rows of equal logits, many times: id 0."""
    torch = g._torch
    x = torch.full((64, 262144), 1.5, device=g.torch_device)
    u, t = torch.zeros(64, dtype=torch.float64, device=g.torch_device), torch.zeros(64, device=g.torch_device)
    for _ in range(50):
        assert not g.sample_requests(x, t, uniforms=u).any()
    x[:, 77777:] = 1.75
    for _ in range(50):
        assert bool((g.sample_requests(x, t, uniforms=u) == 77777).all())
