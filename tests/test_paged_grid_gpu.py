"""How gq_paged_attention spreads its work over the GPU (needs a B200)."""
import json

import numpy as np
import pytest

from gq import CudaBackend, _abi

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def g():
    be = CudaBackend(0)
    yield be
    be.close()


@pytest.mark.parametrize("name,d,ps", [("bfloat16", 96, 16), ("float8_e4m3fn", 64, 16), ("float32", 128, 24)])
def test_rows_without_tiles_fill_the_gpu(g, name, d, ps, tmp_path):
    """The kernel of the head_dims and page sizes that have no tiles hides its loads' latency
    by warps: four CTAs per SM where there is work for them (two took 1.6-1.8 times as long)."""
    from torch.profiler import ProfilerActivity, profile
    torch = g._torch
    n = 5000
    pages_each = -(-n // ps)
    k, v = (torch.randn(2 * pages_each, 1, ps, d, device=g.torch_device).to(getattr(torch, name)) for _ in range(2))
    table = torch.arange(2 * pages_each, dtype=torch.int32, device=g.torch_device).view(2, pages_each)
    lens = torch.tensor([n] * 2, dtype=torch.int32, device=g.torch_device)
    # units of four blocks of 8 query heads: 2 x 4 x 79 tiles of 64 keys
    q = torch.randn(2, 32, d, device=g.torch_device)
    pages = g.kv_pages(k, v)
    g.paged_attention(pages, q, table, lens, scale=0.1)
    torch.cuda.synchronize()
    with profile(activities=[ProfilerActivity.CUDA]) as prof:
        g.paged_attention(pages, q, table, lens, scale=0.1)
        torch.cuda.synchronize()
    assert g.lib.gq_sync(g.ctx) == _abi.GQ_OK
    path = tmp_path / "trace.json"
    prof.export_chrome_trace(str(path))
    grids = [e["args"]["grid"] for e in json.loads(path.read_text())["traceEvents"]
             if "paged_rows_kernel" in e.get("name", "") and "grid" in e.get("args", {})]
    assert [int(np.prod(x)) for x in grids] == [4 * g.num_sms()]
