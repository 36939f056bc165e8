"""Numbers that are none in attention over pages of f32, f16, bf16 and e4m3 (needs a B200): a NaN in a query or a visible
key is in the result, however the request is cut."""
import numpy as np
import pytest

from gq import CudaBackend
from numerics import rel_l2
from test_e2m1_pages_gpu import ATTN_REL_L2, attention_ref, dev

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def g():
    be = CudaBackend(0)
    yield be
    be.close()


# clusters of 8 and less, of 1, requests that are cut, and the kernel without tiles
@pytest.mark.parametrize("lens,dim,hq,hkv,ps", [([333], 256, 8, 1, 16), ([200], 512, 8, 1, 64), ([300, 200], 128, 8, 2, 32),
                                                ([150] * 300, 64, 4, 1, 16), ([5000, 300], 256, 8, 1, 16), ([500, 40], 48, 4, 2, 16)])
@pytest.mark.parametrize("typ", ["f32", "f16", "bf16", "e4m3"])
@pytest.mark.parametrize("where", ["query", "first keys", "last keys", "one key"])
def test_nan_is_not_lost(g, typ, lens, dim, hq, hkv, ps, where):
    torch = g._torch
    rng = np.random.default_rng(dim + len(lens))
    lens = np.array(lens, np.int32)
    need = -(-lens // ps)
    pages = int(need.sum())
    dt = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "e4m3": torch.float8_e4m3fn}[typ]
    pool = [torch.from_numpy(rng.standard_normal((pages, hkv, ps, dim)).astype(np.float32)).to(dt) for _ in range(2)]
    table = np.zeros((len(lens), int(need.max())), np.int32)
    table[np.arange(table.shape[1])[None] < need[:, None]] = rng.permutation(pages)
    q = rng.standard_normal((len(lens), hq, dim)).astype(np.float32)
    n, group = int(lens[0]), hq // hkv
    bad = np.zeros((len(lens), hq, dim), bool)
    keys = pool[0].float()
    if where == "query":
        q[0, hq - 1, 3] = np.nan
        bad[0, hq - 1] = True
    else:
        few = min(128, n // 2)
        at = dict(zip(("first keys", "last keys", "one key"), (np.arange(few), np.arange(n - few, n), np.array([n // 2]))))[where]
        keys[table[0, at // ps], hkv - 1, at % ps] = float("nan")
        bad[0, hq - group:] = True
    k, v = keys.to(dt).to(g.torch_device), pool[1].to(g.torch_device)
    out = g.paged_attention(g.kv_pages(k, v), dev(g, q), dev(g, table), dev(g, lens), scale=dim ** -0.5)
    got = out.data.cpu().numpy().reshape(bad.shape)
    assert np.isnan(got[bad]).all()
    clean = lambda x: np.where(np.isnan(x), 0.0, x)  # noqa: E731
    want = attention_ref(clean(q), clean(keys.double().numpy()), pool[1].double().numpy(), table, lens, dim ** -0.5, 0, 0.0, ps)
    assert rel_l2(got[~bad], want.reshape(bad.shape)[~bad]) <= ATTN_REL_L2
