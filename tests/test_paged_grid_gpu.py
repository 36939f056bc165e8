"""How gq_paged_attention spreads its work over the GPU (needs a B200)."""
import json
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "gemma-4-webgpu-kernels_b200")


def grids(path):
    """A process of its own (a profiler's sessions in one process can lose launches): the
    grids of the kernel over a float8, a bfloat16 and a float32 cache."""
    import torch
    from torch.profiler import ProfilerActivity, profile

    from gq import CudaBackend, _abi
    g, n = CudaBackend(0), 5000
    calls = []
    for name, d, ps in (("float8_e4m3fn", 64, 16), ("bfloat16", 96, 16), ("float32", 128, 24)):
        each = -(-n // ps)
        k, v = (torch.randn(2 * each, 1, ps, d, device=g.torch_device).to(getattr(torch, name)) for _ in range(2))
        table = torch.arange(2 * each, dtype=torch.int32, device=g.torch_device).view(2, each)
        lens = torch.tensor([n] * 2, dtype=torch.int32, device=g.torch_device)
        # 32 query heads are four units of 8: 2 x 4 x 79 tiles of 64 keys
        calls.append((g.kv_pages(k, v), torch.randn(2, 32, d, device=g.torch_device), table, lens))
    run = lambda: [g.paged_attention(*c, scale=0.1) for c in calls]  # noqa: E731
    run()
    torch.cuda.synchronize()
    with profile(activities=[ProfilerActivity.CUDA]) as prof:
        run()
        torch.cuda.synchronize()
    assert g.lib.gq_sync(g.ctx) == _abi.GQ_OK
    prof.export_chrome_trace(path)
    with open(path) as f:
        events = [e for e in json.load(f)["traceEvents"] if "paged_rows_kernel" in e.get("name", "") and "grid" in e.get("args", {})]
    print(json.dumps({"sms": g.num_sms(), "grids": [e["args"]["grid"] for e in events]}))


def test_rows_without_tiles_fill_the_gpu(tmp_path):
    """The kernel of the head_dims and page sizes that have no tiles hides its loads' latency
    by warps: four CTAs per SM where there is work for them (two took 1.6-1.8 times as long)."""
    out = subprocess.run([sys.executable, os.path.abspath(__file__), str(tmp_path / "trace.json")], capture_output=True,
                         text=True, timeout=300, env={**os.environ, "PYTHONPATH": PKG})
    assert out.returncode == 0, out.stderr[-2000:]
    got = json.loads(out.stdout.strip().splitlines()[-1])
    assert got["grids"] == [[4 * got["sms"], 1, 1]] * 3


if __name__ == "__main__":
    grids(sys.argv[1])
