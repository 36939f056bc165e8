"""Numbers that are none in attention over pages of 4-bit values (needs a B200): a NaN in a query, a visible key or a
visible value is in the result, however the request is cut."""
import numpy as np
import pytest

import e2m1_ref as ref
from gq import CudaBackend
from numerics import rel_l2
from test_e2m1_pages_gpu import ATTN_REL_L2, attention_ref, dev, pools_of

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def g():
    be = CudaBackend(0)
    yield be
    be.close()


# one request in a cluster of 8 and less, one in clusters of 1, several that are cut, and the kernel without tiles
SIZES = [([333], 256, 8, 1, 16), ([77], 512, 8, 1, 64), ([300, 200], 128, 8, 2, 32), ([150] * 300, 64, 4, 1, 16),
         ([5000, 300], 256, 8, 1, 16), ([9000], 128, 16, 2, 64), ([500, 40], 48, 4, 2, 16)]


@pytest.mark.parametrize("lens,dim,hq,hkv,ps", SIZES)
@pytest.mark.parametrize("where", ["query", "first keys", "last keys", "one key", "value"])
def test_nan_is_not_lost(g, lens, dim, hq, hkv, ps, where):
    rng = np.random.default_rng(dim + len(lens))
    lens = np.array(lens, np.int32)
    need = -(-lens // ps)
    k, v = pools_of(rng, int(need.sum()), hkv, ps, dim)
    table = np.zeros((len(lens), int(need.max())), np.int32)
    table[np.arange(table.shape[1])[None] < need[:, None]] = rng.permutation(int(need.sum()))
    q = rng.standard_normal((len(lens), hq, dim)).astype(np.float32)
    n, group = int(lens[0]), hq // hkv  # request 0 has it, and of its heads the last or the last key-value head's
    bad = np.zeros((len(lens), hq, dim), bool)
    if where == "query":
        q[0, hq - 1, 3] = np.nan
        bad[0, hq - 1] = True
    elif where == "value":
        j = n // 3
        v[table[0, j // ps], hkv - 1, j % ps, dim // 2] = 0x7f  # the first block's scale
        bad[0, hq - group:, :16] = True
    else:
        few = min(64, n // 2)
        at = dict(zip(("first keys", "last keys", "one key"), (np.arange(few), np.arange(n - few, n), np.array([n // 2]))))[where]
        k[table[0, at // ps], hkv - 1, at % ps, dim // 2:] = 0x7f
        bad[0, hq - group:] = True
    out = g.paged_attention(g.kv_pages(dev(g, k), dev(g, v), 1 / 32, 1 / 32), dev(g, q), dev(g, table), dev(g, lens), scale=dim ** -0.5)
    got = out.data.cpu().numpy().reshape(bad.shape)
    assert np.isnan(got[bad]).all()
    clean = lambda x: np.where(np.isnan(x), 0.0, x)  # noqa: E731
    want = attention_ref(clean(q), clean(ref.decode(k, 1 / 32)), clean(ref.decode(v, 1 / 32)), table, lens, dim ** -0.5, 0, 0.0, ps)
    assert rel_l2(got[~bad], want.reshape(bad.shape)[~bad]) <= ATTN_REL_L2


@pytest.mark.parametrize("lens,dim,hq,hkv,ps", SIZES)
def test_nan_that_is_not_visible_is_not_seen(g, lens, dim, hq, hkv, ps):
    """The same in keys ahead of the window and behind the length."""
    rng = np.random.default_rng(dim)
    lens = np.array(lens, np.int32)
    need, window = -(-lens // ps) + 1, 37
    k, v = pools_of(rng, int(need.sum()), hkv, ps, dim)
    table = np.arange(int(need.sum()), dtype=np.int32)
    table = np.stack([np.pad(table[e - c:e], (0, int(need.max()) - c)) for c, e in zip(need, np.cumsum(need))])
    q = rng.standard_normal((len(lens), hq, dim)).astype(np.float32)
    kd, vd = ref.decode(k, 1 / 32), ref.decode(v, 1 / 32)
    for b, n in enumerate(lens):
        at = np.r_[0:max(0, n - window), n:need[b] * ps]
        k[table[b, at // ps], :, at % ps] = 255
        v[table[b, at // ps], :, at % ps] = 255
    out = g.paged_attention(g.kv_pages(dev(g, k), dev(g, v), 1 / 32, 1 / 32), dev(g, q), dev(g, table), dev(g, lens), scale=dim ** -0.5,
                            sliding_window=window)
    want = attention_ref(q, kd, vd, table, lens, dim ** -0.5, window, 0.0, ps)
    assert rel_l2(out.data.cpu().numpy(), want) <= ATTN_REL_L2
