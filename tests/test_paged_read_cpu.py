"""CudaBackend.paged_read without a device: pages that the library refuses get as far as the library."""
import pytest
import torch

from gq import CudaBackend, GqError, _abi


@pytest.mark.parametrize("shape", [(4, 1, 16, 0), (4, 2, 16, 0), (4, 0, 16, 64)])
def test_rows_of_no_values(shape):
    g = CudaBackend.__new__(CudaBackend)
    g._torch, g.torch_device, g.ctx, g.device = torch, torch.device("cpu"), None, -1
    seen = []
    g.lib = type("Lib", (), {"gq_paged_read": lambda self, *a: seen.append(a) or _abi.GQ_ERR_INVALID_ARGUMENT})()

    def check(rc, what):
        raise GqError(rc, what)

    g._check = check
    with pytest.raises(GqError) as e:
        g.paged_read(g.kv_pages(torch.zeros(shape), torch.zeros(shape)), torch.zeros(5, dtype=torch.int64))
    assert e.value.status == _abi.GQ_ERR_INVALID_ARGUMENT and len(seen) == 1
