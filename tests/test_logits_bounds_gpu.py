"""gq_process_logits at the bounds of its inputs (needs a B200). The results must equal
the definition: every operation rounds once in f32 on both sides."""
import numpy as np
import pytest

from gq import CudaBackend, GqError, _abi
from test_logits_gpu import dev

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def g():
    be = CudaBackend(0)
    yield be
    be.close()


@pytest.mark.parametrize("offsets,rows", [
    ([0, 10 ** 6, 2, 10 ** 9], [(0, 3), (3, 2), (2, 3)]),
    ([-5, 2, -7, 3], [(0, 2), (2, 0), (0, 3)]),
    ([2 ** 31 - 1, -2 ** 31, 2 ** 31 - 1, 1], [(3, 0), (0, 3), (3, 1)])])
def test_bias_offsets_are_cut_to_the_entries(g, offsets, rows):
    """rows: the entries that are left of each row's."""
    torch = g._torch
    x = np.random.default_rng(1).standard_normal((3, 100)).astype(np.float32)
    ids, values = [5, 7, 99], [1.5, -2.25, 30.0]
    got = g.process_logits(dev(g, x, np.float32), bias_ids=dev(g, ids, np.int32), bias_values=dev(g, values, np.float32),
                           bias_offsets=dev(g, offsets, np.int32)).data
    assert g.lib.gq_sync(g.ctx) == _abi.GQ_OK
    want = x.copy()
    for r, (lo, hi) in enumerate(rows):
        for i in range(lo, hi):
            want[r, ids[i]] += np.float32(values[i])
    np.testing.assert_array_equal(got.cpu().numpy(), want)
    # without the number of entries the last offset says how many there are
    t = [dev(g, x, np.float32), dev(g, ids, np.int32), dev(g, values, np.float32), dev(g, offsets[:3] + [3], np.int32)]
    y = torch.empty(3, 100, device=g.torch_device)
    rc = g.lib.gq_process_logits(g.ctx, t[0].data_ptr(), 3, 100, 0, None, 0, None, None, None, t[1].data_ptr(), t[2].data_ptr(),
                                 t[3].data_ptr(), None, 0, 0, None, y.data_ptr(), 0)
    assert rc == _abi.GQ_OK and g.lib.gq_sync(g.ctx) == _abi.GQ_OK
    cut = [min(max(o, 0), 3) for o in offsets[:3]] + [3]
    want = x.copy()
    for r in range(3):
        for i in range(cut[r], cut[r + 1]):
            want[r, ids[i]] += np.float32(values[i])
    np.testing.assert_array_equal(y.cpu().numpy(), want)
    assert g.lib.gq_process_logits_bounded(g.ctx, t[0].data_ptr(), 3, 100, 0, None, 0, None, None, None, t[1].data_ptr(),
                                           t[2].data_ptr(), t[3].data_ptr(), -1, None, 0, 0, None, y.data_ptr(),
                                           0) == _abi.GQ_ERR_INVALID_ARGUMENT


def test_biases_need_all_three_tensors(g):
    x = g._torch.zeros(2, 64, device=g.torch_device)
    all3 = dict(bias_ids=dev(g, [1], np.int32), bias_values=dev(g, [1], np.float32), bias_offsets=dev(g, [0, 1, 1], np.int32))
    for left_out in [("bias_ids",), ("bias_values",), ("bias_offsets",), ("bias_ids", "bias_values"), ("bias_values", "bias_offsets"),
                     ("bias_ids", "bias_offsets")]:
        with pytest.raises(GqError) as e:
            g.process_logits(x, **{k: v for k, v in all3.items() if k not in left_out})
        assert e.value.status == _abi.GQ_ERR_INVALID_ARGUMENT
    assert g.process_logits(x, **all3).data[0, 1] == 1.0
    none = dict(bias_ids=dev(g, [], np.int32), bias_values=dev(g, [], np.float32), bias_offsets=dev(g, [0, 0, 0], np.int32))
    assert (g.process_logits(x, **none).data == 0).all()
