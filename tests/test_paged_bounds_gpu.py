"""The paged-cache calls at the bounds of their arguments (needs a B200)."""
import numpy as np
import pytest

from gq import CudaBackend, GqError, _abi

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def g():
    be = CudaBackend(0)
    yield be
    be.close()


def i32(g, a):
    return g._torch.tensor(np.asarray(a, dtype=np.int32), device=g.torch_device)


def test_scales_whose_reciprocal_overflows_are_refused(g):
    """1 / 1e-39 is an infinity: zeros would be stored as NaN, everything else as the largest
    code."""
    torch = g._torch
    z = lambda: torch.zeros(2, 1, 16, 128, device=g.torch_device).to(torch.float8_e4m3fn)  # noqa: E731
    rows, slots = torch.ones(1, 1, 128, device=g.torch_device), torch.zeros(1, dtype=torch.int64, device=g.torch_device)
    for scales in ((1e-39, 1.0), (1.0, 1e-39)):
        pages = g.kv_pages(z(), z(), *scales)
        for call in (lambda: g.paged_append(pages, rows, rows, slots),
                     lambda: g.paged_attention(pages, rows, i32(g, [[0]]), i32(g, [1]))):
            with pytest.raises(GqError) as e:
                call()
            assert e.value.status == _abi.GQ_ERR_INVALID_ARGUMENT
    smallest = float(np.float32(2.0 ** -126))
    pages = g.kv_pages(z(), z(), smallest, smallest)
    g.paged_append(pages, rows * smallest, rows * smallest, slots)
    assert g.lib.gq_sync(g.ctx) == _abi.GQ_OK and (pages.k[0, 0, 0].float() == 1.0).all()
