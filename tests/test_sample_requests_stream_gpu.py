"""gq_sample_requests into new tokens, on a backend with a stream of its own (needs a B200)."""
import pytest

from gq import CudaBackend

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def g():
    be = CudaBackend(0, own_stream=True)
    yield be
    be.close()


def test_tokens_that_torch_still_uses(g):
    """New tokens are written after what torch's stream does with memory that the caller let go of."""
    torch = g._torch
    x = torch.randn(37, 5000, device=g.torch_device)
    u, t = torch.zeros(37, dtype=torch.float64, device=g.torch_device), torch.zeros(37, device=g.torch_device)
    busy = torch.randn(4096, 4096, device=g.torch_device)
    want = x.argmax(1).tolist()
    torch.cuda.synchronize()
    for _ in range(5):
        tokens = g.sample_requests(x, t, uniforms=u)
        g.flush()
        for _ in range(20):
            busy = busy @ busy * 1e-2
        copy = tokens + 1
        tokens.fill_(-7)
        del tokens
        g.begin_frame()
        some = [g.sample_requests(x, t, uniforms=u) for _ in range(64)]  # one of them in that memory
        g.flush()
        torch.cuda.synchronize()
        assert all(tokens.tolist() == want for tokens in some) and (copy - 1).tolist() == want
        del some
