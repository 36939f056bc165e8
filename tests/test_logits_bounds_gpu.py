"""gq_process_logits at the bounds of its inputs (needs a B200). The results must equal
the definition: every operation rounds once in f32 on both sides."""
import numpy as np
import pytest

from gq import CudaBackend, GqError, _abi
from test_logits_gpu import dev, history, reference, run, some_bias

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


# Shapes whose rows are cut into chunks of 16384 columns (those of test_logits_gpu.py give
# chunks of 2048, all but one).


@pytest.mark.parametrize("m,v", [(7, 131077), (40, 16387), (75, 8192), (3, 262144), (40, 16383)])
@pytest.mark.parametrize("place", ["new", "in place", "other phase"])
def test_large_chunks_with_everything(g, m, v, place):
    assert m * -(-v // 4096) >= g.num_sms()
    rng = np.random.default_rng(v + m)
    x = rng.standard_normal((m, v)).astype(np.float32) * 4
    words = -(-v // 32)
    masks = rng.integers(0, 2 ** 32, (m + 2, words), dtype=np.uint32) | rng.integers(0, 2 ** 32, (m + 2, words), dtype=np.uint32)
    masks[1] = 0  # a row with nothing allowed
    mask_rows = rng.integers(-1, m + 3, m)
    mask_rows[0] = 1
    kw = dict(history(rng, m, v, 700), bias=some_bias(rng, m, v, 40), masks=masks, mask_rows=mask_rows)
    got = run(g, x, place=place, lead=v % 4, ld=v + 3 if v % 2 else v, **kw)
    np.testing.assert_array_equal(got, reference(x, **kw))


@pytest.mark.parametrize("what", ["tokens", "bias", "masks", "nothing"])
def test_large_chunks_each_step_alone(g, what):
    rng = np.random.default_rng(3)
    m, v = 13, 50001
    assert m * -(-v // 4096) >= g.num_sms()
    x = rng.standard_normal((m, v)).astype(np.float32)
    kw = {}
    if what == "tokens":
        kw = history(rng, m, v, 5000)
    elif what == "bias":
        kw = dict(bias=some_bias(rng, m, v, 2000))
    elif what == "masks":
        kw = dict(masks=rng.integers(0, 2 ** 32, (m, -(-v // 32)), dtype=np.uint32))
    np.testing.assert_array_equal(run(g, x, **kw), reference(x, **kw))


@pytest.mark.parametrize("v,lead", [(16387, 0), (16387, 1), (40960, 0)])
def test_more_seen_tokens_than_a_chunks_list(g, v, lead):
    """9000 different ids in the first 16384 columns: more than the 2048 that a CTA lists, so
    it looks at every column."""
    rng = np.random.default_rng(v + lead)
    m, n, f = 40, 12000, np.float32
    x = rng.standard_normal((m, v)).astype(np.float32) * 4
    tokens = np.stack([np.concatenate([rng.permutation(16384)[:9000], rng.integers(0, v, n - 9000)]) for _ in range(m)])
    lens = np.full(m, n)
    lens[1:] = rng.integers(0, n + 1, m - 1)
    prompt = (lens * rng.random(m)).astype(np.int64)
    pen = np.stack([1 + rng.random(m), rng.random(m), rng.random(m) * 0.2], 1).astype(f)
    masks = rng.integers(0, 2 ** 32, (m, -(-v // 32)), dtype=np.uint32) | rng.integers(0, 2 ** 32, (m, -(-v // 32)), dtype=np.uint32)
    kw = dict(bias=some_bias(rng, m, v, 60), masks=masks)
    y = x.copy()
    for r in range(m):
        ids = tokens[r, :lens[r]]
        seen, made = np.bincount(ids, minlength=v) > 0, np.bincount(ids[prompt[r]:], minlength=v)
        y[r] = np.where(seen, np.where(y[r] > 0, y[r] / pen[r, 0], y[r] * pen[r, 0]), y[r])
        y[r] = np.where(made > 0, (y[r] - pen[r, 2] * made.astype(f)) - pen[r, 1], y[r])
    assert y.dtype == f
    got = run(g, x, tokens=tokens, prompt=prompt, lens=lens, pen=pen, lead=lead, **kw)
    np.testing.assert_array_equal(got, reference(y, **kw))
