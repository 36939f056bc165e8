"""CudaBackend.kv_pages describes a pool on the host: what it hands to the library, and
what it refuses, without a device (a backend whose device is the CPU, and no context)."""
import pytest
import torch

from gq import CudaBackend, GqError, _abi


@pytest.fixture
def g():
    be = CudaBackend.__new__(CudaBackend)
    be._torch, be.torch_device, be.ctx = torch, torch.device("cpu"), None
    return be


def test_strides_of_pages(g):
    pool = torch.zeros(6, 2, 3, 16, 64)
    for k, v, apart in ((pool[:, 0], pool[:, 1], 2 * 3 * 16 * 64), (pool[:, 0].contiguous(), pool[:, 1].contiguous(), 3 * 16 * 64),
                        (pool[:1, 0], pool[:1, 1], 3 * 16 * 64), (pool[:0, 0], pool[:0, 1], 3 * 16 * 64)):
        st = g.kv_pages(k, v).struct
        assert (st.n_pages, st.page_size, st.heads, st.head_dim, st.page_stride) == (k.shape[0], 16, 3, 64, apart)


def test_pages_that_share_memory_are_refused(g):
    """One page expanded to many has stride 0, which means packed pages to the library: it
    would read and write past the page."""
    one = torch.zeros(1, 3, 16, 64)
    for k in (one.expand(6, 3, 16, 64), torch.zeros(20000).as_strided((6, 3, 16, 64), (64, 1024, 64, 1))):
        with pytest.raises(GqError) as e:
            g.kv_pages(k, k)
        assert e.value.status == _abi.GQ_ERR_INVALID_ARGUMENT


def test_append_refuses_rows_by_head(g):
    """[heads, T, head_dim] holds as many values as [T, heads, head_dim], in another order."""
    calls = []
    g.device, g.lib = -1, type("Lib", (), {"gq_paged_append": lambda self, *a: calls.append(a) or 0})()
    pages = g.kv_pages(torch.zeros(4, 2, 16, 64), torch.zeros(4, 2, 16, 64))
    ok, slots = torch.zeros(5, 2, 64), torch.zeros(5, dtype=torch.int64)
    for rows in (ok, ok.view(5, 128), ok.view(-1), ok[None], torch.zeros(5, 256)[:, :128]):
        g.paged_append(pages, rows, ok, slots)
    assert len(calls) == 5
    by_head = torch.zeros(2, 5, 64)
    for k, v in ((by_head, ok), (ok, by_head)):
        with pytest.raises(GqError) as e:
            g.paged_append(pages, k, v, slots)
        assert e.value.status == _abi.GQ_ERR_INVALID_ARGUMENT
    assert len(calls) == 5
