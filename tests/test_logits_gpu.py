"""gq_process_logits against the definition, row by row (needs a B200).

Every operation rounds once in f32 on both sides (a division, a product, a
subtraction, a sum), so the results must be equal.
"""
import numpy as np
import pytest

from gq import CudaBackend, GqError, _abi

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def g():
    be = CudaBackend(0)
    yield be
    be.close()


def dev(g, a, dtype):
    return g._torch.tensor(np.asarray(a, dtype=dtype), device=g.torch_device)


def reference(x, tokens=None, prompt=None, lens=None, pen=None, bias=None, masks=None, mask_rows=None):
    y = np.array(x, dtype=np.float32)
    m, v = y.shape
    f = np.float32
    for r in range(m):
        if tokens is not None:
            n = min(int(lens[r]), tokens.shape[1])
            row = [int(t) for t in tokens[r, :max(n, 0)]]
            for c in {t for t in row if 0 <= t < v}:
                y[r, c] = y[r, c] / f(pen[r, 0]) if y[r, c] > 0 else y[r, c] * f(pen[r, 0])
                made = sum(1 for i, t in enumerate(row) if t == c and i >= prompt[r])
                if made:
                    y[r, c] = (y[r, c] - f(pen[r, 2]) * f(made)) - f(pen[r, 1])
        if bias is not None:
            for c, b in dict(bias[r]).items():  # the last entry of an id counts
                if 0 <= c < v:
                    y[r, c] = y[r, c] + f(b)
        if masks is not None:
            k = int(mask_rows[r]) if mask_rows is not None else r
            if 0 <= k < len(masks):
                bits = np.unpackbits(masks[k].view(np.uint8), bitorder="little")[:v]
                y[r, bits == 0] = -np.inf
    return y


def run(g, x, tokens=None, prompt=None, lens=None, pen=None, bias=None, masks=None, mask_rows=None, ld=None, lead=0, place="new"):
    torch = g._torch
    m, v = x.shape
    ld = ld or v
    buf = torch.full((m * ld + lead + 8,), 77.0, device=g.torch_device)
    lg = buf[lead:lead + m * ld].view(m, ld)[:, :v]
    lg.copy_(dev(g, x, np.float32))
    kw = {}
    if tokens is not None:
        kw.update(tokens=dev(g, tokens, np.int32), prompt_lens=dev(g, prompt, np.int32), lens=dev(g, lens, np.int32),
                  penalties=dev(g, pen, np.float32))
    if bias is not None:
        flat = [e for row in bias for e in row]
        kw.update(bias_ids=dev(g, [c for c, _ in flat], np.int32), bias_values=dev(g, [b for _, b in flat], np.float32),
                  bias_offsets=dev(g, np.cumsum([0] + [len(row) for row in bias]), np.int32))
    if masks is not None:
        kw["masks"] = dev(g, masks.view(np.int32), np.int32)
        if mask_rows is not None:
            kw["mask_rows"] = dev(g, mask_rows, np.int32)
    if place == "in place":
        out = lg
    elif place == "other phase":  # an output on another phase of a 16-byte boundary
        out = torch.full((m * ld + 16,), 55.0, device=g.torch_device)[lead + 1:lead + 1 + m * ld].view(m, ld)[:, :v]
    else:
        out = torch.full((m, v), 55.0, device=g.torch_device)
    g.process_logits(lg, out=out, **kw)
    assert g.lib.gq_sync(g.ctx) == _abi.GQ_OK
    if ld > v and place == "in place":
        assert (buf[lead:lead + m * ld].view(m, ld)[:, v:] == 77.0).all(), "wrote past the rows"
    return out.cpu().numpy()


def history(rng, m, v, n):
    tokens = (rng.random((m, n)) ** 3 * v).astype(np.int64)
    tokens[rng.random((m, n)) < 0.05] = v + 3  # ids past the vocabulary, and none
    tokens[rng.random((m, n)) < 0.05] = -1
    lens = rng.integers(0, n + 1, m)
    lens[0] = n
    prompt = (lens * rng.random(m)).astype(np.int64)
    pen = np.stack([1 + rng.random(m), rng.random(m) - 0.3, rng.random(m) - 0.3], 1).astype(np.float32)
    return dict(tokens=tokens, prompt=prompt, lens=lens, pen=pen)


def some_bias(rng, m, v, n):
    return [[(int(c), float(b)) for c, b in zip(rng.integers(-2, v + 2, k), rng.standard_normal(k) * 5)]
            for k in rng.integers(0, n + 1, m)]


@pytest.mark.parametrize("m,v", [(1, 1), (1, 31), (3, 33), (2, 8192), (5, 8193), (2, 65535), (1, 65541), (3, 131077), (1, 262144)])
@pytest.mark.parametrize("place", ["new", "in place", "other phase"])
def test_everything_together(g, m, v, place):
    rng = np.random.default_rng(v + m)
    x = rng.standard_normal((m, v)).astype(np.float32) * 4
    masks = rng.integers(0, 2 ** 32, (m, -(-v // 32)), dtype=np.uint32) | rng.integers(0, 2 ** 32, (m, -(-v // 32)), dtype=np.uint32)
    kw = dict(history(rng, m, v, 700), bias=some_bias(rng, m, v, 40), masks=masks)
    got = run(g, x, place=place, lead=v % 4, ld=v + 3 if v % 2 else v, **kw)
    np.testing.assert_array_equal(got, reference(x, **kw))


@pytest.mark.parametrize("what", ["tokens", "bias", "masks", "nothing"])
def test_each_step_alone(g, what):
    rng = np.random.default_rng(3)
    m, v = 4, 50000
    x = rng.standard_normal((m, v)).astype(np.float32)
    kw = {}
    if what == "tokens":
        kw = history(rng, m, v, 5000)
    elif what == "bias":
        kw = dict(bias=some_bias(rng, m, v, 2000))
    elif what == "masks":
        kw = dict(masks=rng.integers(0, 2 ** 32, (3, -(-v // 32)), dtype=np.uint32), mask_rows=np.array([2, -1, 0, 99]))
    np.testing.assert_array_equal(run(g, x, **kw), reference(x, **kw))


def test_long_history_of_few_tokens(g):
    """100,000 repeats of a handful of ids: counts far past 16 bits."""
    rng = np.random.default_rng(8)
    v, n = 300000, 100000
    tokens = rng.choice([0, 5, 8191, 8192, 65535, 65536, v - 1], (2, n))
    kw = dict(tokens=tokens, prompt=np.array([0, 50000]), lens=np.array([n, n + 5]),  # a length past the row is cut to it
              pen=np.array([[1.3, 0.5, 0.001], [2.0, -0.5, 0.01]], np.float32))
    x = rng.standard_normal((2, v)).astype(np.float32)
    np.testing.assert_array_equal(run(g, x, **kw), reference(x, **kw))


def test_rows_with_nothing_allowed_and_nonfinite_values(g):
    v = 100
    x = np.zeros((4, v), np.float32)
    x[0, :4] = [np.inf, -np.inf, np.nan, -0.0]
    x[1] = np.finfo(np.float32).min
    masks = np.zeros((4, 4), np.uint32)
    masks[0] = 0xFFFFFFFF
    masks[3, 1] = 1  # column 32 alone
    bias = [[(5, np.inf), (6, -np.inf)], [], [(7, np.inf)], [(7, np.inf), (32, 1.0), (32, 2.0)]]
    pen = np.array([[1.5, 0.1, 0.1]] * 4, np.float32)
    kw = dict(tokens=np.tile(np.arange(10), (4, 1)), prompt=np.zeros(4, int), lens=np.full(4, 10), pen=pen, bias=bias, masks=masks)
    got = run(g, x, **kw)
    np.testing.assert_array_equal(got, reference(x, **kw))
    assert (got[2] == -np.inf).all() and np.isfinite(got[3]).sum() == 1 and got[3, 32] == 2.0


def test_refusals(g):
    torch = g._torch
    x = torch.zeros(2, 64, device=g.torch_device)
    tok = dev(g, np.zeros((2, 3)), np.int32)
    ln, pen = dev(g, [1, 1], np.int32), torch.ones(2, 3, device=g.torch_device)
    for kw in (dict(tokens=tok), dict(tokens=tok, prompt_lens=ln, lens=ln[:1], penalties=pen),
               dict(tokens=tok.long(), prompt_lens=ln, lens=ln, penalties=pen),
               dict(tokens=tok, prompt_lens=ln, lens=ln, penalties=pen[:1]),
               dict(masks=dev(g, np.zeros((2, 1)), np.int32)), dict(masks=dev(g, np.zeros((1, 2)), np.int32)),
               dict(bias_ids=dev(g, [1], np.int32), bias_values=torch.ones(1, device=g.torch_device), bias_offsets=ln),
               dict(out=torch.zeros(2, 65, device=g.torch_device))):
        with pytest.raises(GqError) as e:
            g.process_logits(x, **kw)
        assert e.value.status == _abi.GQ_ERR_INVALID_ARGUMENT
    with pytest.raises(GqError):
        g.process_logits(x[:1].expand(2, 64))
    assert g.lib.gq_process_logits(None, *([None] + [0] * 3 + [None, 0] + [None] * 7 + [0, 0, None, None, 0])) == \
        _abi.GQ_ERR_INVALID_ARGUMENT
    assert g.lib.gq_process_logits(g.ctx, x.data_ptr(), 1, 1 << 28, 0, None, 0, None, None, None, None, None, None, None, 0,
                                   0, None, x.data_ptr(), 0) == _abi.GQ_ERR_UNSUPPORTED
    assert g.process_logits(torch.zeros(0, 64, device=g.torch_device)).data.shape == (0, 64)
    assert g.lib.gq_sync(g.ctx) == _abi.GQ_OK
