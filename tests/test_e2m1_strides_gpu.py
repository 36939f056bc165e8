"""Pages of 4-bit values any number of bytes apart (needs a B200): append, read and attention."""
import numpy as np
import pytest

import e2m1_ref as ref
from gq import CudaBackend
from numerics import rel_l2
from test_e2m1_pages_gpu import ATTN_REL_L2, attention_ref, dev, hard_rows, pools_of

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def g():
    be = CudaBackend(0)
    yield be
    be.close()


def apart(g, pages, heads, ps, row, more):
    """Two pools whose pages lie `more` bytes apart, and what lies in between (all 3)."""
    torch = g._torch
    page = heads * ps * row
    n = -(-pages * (page + more) // 16) * 16
    store = torch.full((2, n), 3, dtype=torch.uint8, device=g.torch_device)
    views = [s.as_strided((pages, heads, ps, row), (page + more, ps * row, row, 1), s.storage_offset()) for s in (store[0], store[1])]
    assert all(t.data_ptr() % 16 == 0 for t in views)
    return store, views


@pytest.mark.parametrize("heads,dim,ps", [(1, 64, 16), (1, 512, 16), (2, 128, 32), (3, 256, 8), (2, 48, 7)])
@pytest.mark.parametrize("more", [1, 2, 4, 5, 8, 16, 2304])
def test_pages_any_bytes_apart(g, heads, dim, ps, more):
    torch = g._torch
    rng = np.random.default_rng(dim * 31 + more)
    pages, row = 9, dim // 16 * 9
    store, views = apart(g, pages, heads, ps, row, more)
    pools = pools_of(rng, pages, heads, ps, dim)
    for view, pool in zip(views, pools):
        view.copy_(dev(g, pool))
    desc = g.kv_pages(*views, 1 / 32, 1 / 32)
    assert desc.struct.page_stride == heads * ps * row + more
    # rows written over some of them
    n = pages * ps // 2
    slots = rng.permutation(pages * ps)[:n]
    x = [hard_rows(rng, n, heads * dim) for _ in range(2)]
    with np.errstate(over="ignore"):
        new = [ref.encode(r.reshape(n, heads, dim), 1 / 32) for r in x]
    g.paged_append(desc, dev(g, x[0]), dev(g, x[1]), dev(g, slots))
    k, v = g.paged_read(desc, torch.arange(pages * ps, device=g.torch_device))
    g.flush()
    for pool, r, view, got in zip(pools, new, views, (k, v)):
        pool[slots // ps, :, slots % ps] = r
        assert np.array_equal(view.cpu().numpy(), pool)
        want = ref.decode(pool, 1 / 32).transpose(0, 2, 1, 3).reshape(pages * ps, heads, dim).astype(np.float32)
        assert np.array_equal(got.cpu().numpy(), want, equal_nan=True)
    for i in range(2):  # nothing in between was touched
        between = store[i].clone()
        between.as_strided(views[i].shape, views[i].stride(), between.storage_offset()).fill_(3)
        assert bool((between == 3).all())
    # attention over pages of numbers
    pools = pools_of(rng, pages, heads, ps, dim)
    for view, pool in zip(views, pools):
        view.copy_(dev(g, pool))
    q = rng.standard_normal((2, 4 * heads, dim)).astype(np.float32)
    table, lens = np.array([[3, 0, 4, 1], [8, 7, 2, 2 ** 30]], np.int32), np.array([3 * ps + 2, 2 * ps + 5], np.int32)
    out = g.paged_attention(desc, dev(g, q), dev(g, table), dev(g, lens), scale=0.1)
    want = attention_ref(q, ref.decode(pools[0], 1 / 32), ref.decode(pools[1], 1 / 32), table, lens, 0.1, 0, 0.0, ps)
    assert rel_l2(out.data.cpu().numpy(), want) <= ATTN_REL_L2
