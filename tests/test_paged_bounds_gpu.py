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


@pytest.mark.parametrize("stride", [2 ** 59, 2 ** 60, 2 ** 62])
def test_a_table_stride_past_any_length(g, stride):
    """A row stride whose product with the page size passes 64 bits is as good as any other."""
    torch = g._torch
    gen = torch.Generator(device=g.torch_device).manual_seed(3)
    k, v = (torch.randn(4, 1, 16, 128, generator=gen, device=g.torch_device) for _ in range(2))
    pages, q = g.kv_pages(k, v), torch.randn(1, 8, 128, generator=gen, device=g.torch_device)
    table, lens = i32(g, [[2, 0, 3, 1]]), i32(g, [50])
    want = g.paged_attention(pages, q, table, lens, scale=0.1).data.clone()
    out = torch.zeros(1, 8 * 128, device=g.torch_device)
    rc = g.lib.gq_paged_attention(g.ctx, pages.ref, q.data_ptr(), 1, 8, 0, table.data_ptr(), stride, lens.data_ptr(), 0.1, 0,
                                  0.0, out.data_ptr())
    assert rc == _abi.GQ_OK and g.lib.gq_sync(g.ctx) == _abi.GQ_OK
    # (another cut of the keys: another order of the sums)
    assert float((out - want).norm() / want.norm()) <= 1e-5
    free, keep, count, left, tot = i32(g, [9, 9, 9, 9]), i32(g, [17]), i32(g, [0]), i32(g, [-9]), i32(g, [-9])
    rc = g.lib.gq_paged_release(g.ctx, 1, 16, lens.data_ptr(), keep.data_ptr(), table.data_ptr(), stride, free.data_ptr(), 4,
                                count.data_ptr(), left.data_ptr(), tot.data_ptr())
    assert rc == _abi.GQ_OK and g.lib.gq_sync(g.ctx) == _abi.GQ_OK
    assert free.tolist() == [1, 3, 9, 9] and int(left) == 2 and int(tot) == 17
