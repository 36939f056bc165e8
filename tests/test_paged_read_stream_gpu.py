"""gq_paged_read into new tensors, on a backend with a stream of its own (needs a B200): the rows are there and rows
without a slot are 0, whatever torch's current stream is at, and replayed too."""
import numpy as np
import pytest

import e2m1_ref as ref
from gq import CudaBackend
from test_e2m1_pages_gpu import dev

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def g():
    be = CudaBackend(0, own_stream=True)
    yield be
    be.close()


def some_pages(g, rng, pages=40, ps=16, dim=256):
    pools = [rng.integers(0, 127, (pages, 1, ps, dim // 16 * 9), dtype=np.uint8) for _ in range(2)]
    values = [ref.decode(p, 0.5).astype(np.float32).reshape(pages * ps, 1, dim) for p in pools]
    return g.kv_pages(*(dev(g, p) for p in pools), 0.5, 0.5), values


def expect(values, slots):
    return [np.where((slots >= 0)[:, None, None], x[slots], np.float32(0)) for x in values]


def test_rows_are_not_wiped(g):
    torch = g._torch
    rng = np.random.default_rng(0)
    pages, values = some_pages(g, rng)
    slots = rng.permutation(640)[:500]
    slots[::9] = -1
    d, busy = dev(g, slots), torch.randn(4096, 4096, device=g.torch_device)
    torch.cuda.synchronize()
    for _ in range(5):
        for _ in range(20):
            busy = busy @ busy * 1e-2  # torch's stream is behind
        got = g.paged_read(pages, d)
        g.flush()
        other = torch.cuda.Stream(g.torch_device)  # (not behind the work of torch's stream)
        with torch.cuda.stream(other):
            got = [x.cpu().numpy() for x in got]
        torch.cuda.synchronize()
        for x, want in zip(got, expect(values, slots)):
            assert np.array_equal(x, want)


def test_memory_that_torch_still_uses(g):
    """New tensors are written after what torch's stream does with memory that the caller let go of."""
    torch = g._torch
    rng = np.random.default_rng(1)
    pages, values = some_pages(g, rng)
    slots = rng.permutation(640)[:500]
    d, busy = dev(g, slots), torch.randn(4096, 4096, device=g.torch_device)
    want = expect(values, slots)
    g.paged_read(pages, d)
    g.flush()
    for _ in range(5):
        k, v = g.paged_read(pages, d)
        g.flush()
        for _ in range(20):
            busy = busy @ busy * 1e-2
        sums = k.double() + v.double()  # read late
        k.fill_(-1.0)  # and written
        del k, v
        g.begin_frame()
        k, v = g.paged_read(pages, d)
        g.flush()
        torch.cuda.synchronize()
        assert np.array_equal(k.cpu().numpy(), want[0]) and np.array_equal(v.cpu().numpy(), want[1])
        assert np.array_equal(sums.cpu().numpy(), want[0].astype(np.float64) + want[1])
        del k, v


def test_recorded(g):
    """A recorded read into new tensors makes rows without a slot 0 at each replay."""
    torch = g._torch
    rng = np.random.default_rng(2)
    pages, values = some_pages(g, rng)
    slots = torch.zeros(300, dtype=torch.int64, device=g.torch_device)
    torch.cuda.synchronize()
    out = []
    graph = g.record(lambda: out.extend(g.paged_read(pages, slots)))
    for _ in range(4):
        now = rng.permutation(640)[:300]
        now[rng.random(300) < 0.3] = -1
        slots.copy_(dev(g, now))
        torch.cuda.synchronize()
        g.replay(graph)
        g.flush()
        for x, want in zip(out, expect(values, now)):
            assert np.array_equal(x.cpu().numpy(), want)
    g.destroy_graph(graph)


def test_on_torchs_stream_and_another(g):
    """A backend on torch's stream keeps to it when another one is torch's current."""
    be = CudaBackend(0)
    torch = be._torch
    rng = np.random.default_rng(3)
    pages, values = some_pages(be, rng)
    slots = rng.permutation(640)[:100]
    slots[3] = -1
    d = dev(be, slots)
    torch.cuda.synchronize()
    other = torch.cuda.Stream(be.torch_device)
    with torch.cuda.stream(other):
        got = be.paged_read(pages, d)
    be.flush()
    for x, want in zip(got, expect(values, slots)):
        assert np.array_equal(x.cpu().numpy(), want)
    be.close()
