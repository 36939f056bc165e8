"""The decode step over pages of 4-bit values, with sampling options of each request's own
(gq.paged.PagedDecoder; needs a B200)."""
import numpy as np
import pytest

import e2m1_ref as ref
from gq import CudaBackend, GqError, _abi, e2b, paged
from numerics import rel_l2
from test_e2m1_pages_gpu import ATTN_REL_L2, attention_ref
from test_paged_decode_gpu import rows_of
from test_sample_requests_gpu import sample_ref

pytestmark = pytest.mark.gpu

SCALE = 1 / 32


@pytest.fixture(scope="module")
def g():
    be = CudaBackend(0, own_stream=True)
    yield be
    be.close()


def decoder(g, cfg, weights, lens, sample=(0.0, 0, 1.0), **kw):
    dec = paged.PagedDecoder(g, cfg, weights, len(lens), max_len=96, kv_type="e2m1", k_scale=SCALE, v_scale=SCALE, sample=sample, **kw)
    dec.extend(lens, rows_of(g, cfg, weights, lens), tokens=[[3] * n for n in lens])
    return dec


def splitmix(state):
    z = (state + 0x9e3779b97f4a7c15) % 2 ** 64
    after = z
    z = ((z ^ (z >> 30)) * 0xbf58476d1ce4e5b9) % 2 ** 64
    z = ((z ^ (z >> 27)) * 0x94d049bb133111eb) % 2 ** 64
    return after, ((z ^ (z >> 31)) >> 11) / 2 ** 53


def test_step_over_4_bit_pages(g):
    """What extend stored are the definition's bytes; the last layer's attention is that of its
    query over the stored rows, the step's own among them, before and after recording."""
    torch = g._torch
    cfg = e2b.small_config()
    weights = e2b.Weights(cfg, seed=21)
    lens = [0, 1, 15, 16, 33, 70]
    dec = decoder(g, cfg, weights, lens)
    last = cfg.layers - 1
    src, window = cfg.kv_source(last), cfg.window_of(last)
    for layer in dec.pages:
        at = 0
        want = [x.cpu().numpy() for x in rows_of(g, cfg, weights, lens)(layer)]
        for b, n in enumerate(lens):
            for got, w in zip(dec.rows_of(b)(layer), want):
                x = ref.decode(ref.encode(w[at:at + n].reshape(n, cfg.heads_kv, cfg.dh(layer)), SCALE), SCALE)
                assert np.array_equal(got.cpu().numpy(), x.reshape(n, got.shape[1]).astype(np.float32))
            at += n
    for i in range(4):
        if i == 2:
            dec.record_steps()
        dec.step(np.arange(len(lens)) + 7 * i)
        g.flush()
        now = dec.lens.cpu().numpy()
        assert now.tolist() == [n + i + 1 for n in lens]
        pool = [ref.decode(p.cpu().numpy(), SCALE) for p in (dec.pages[src].k, dec.pages[src].v)]
        q = dec.qr.cpu().numpy().reshape(-1)[:len(lens) * cfg.heads_q * cfg.dh(last)].reshape(len(lens), cfg.heads_q, cfg.dh(last))
        want = attention_ref(q, *pool, dec.table.cpu().numpy(), now, 1.0, window, 0.0, dec.page_size)
        got = dec.attn.cpu().numpy().reshape(-1)[:want.size].reshape(want.shape)
        for b in range(len(lens)):
            assert rel_l2(got[b], want[b]) <= ATTN_REL_L2
        logits = dec.read(dec.logits)
        assert dec.tokens.cpu().numpy().tolist() == np.argmax(logits, 1).tolist()
    dec.close()


@pytest.mark.parametrize("to", ["e2m1", "f32", "e4m3"])
def test_a_request_moves_to_another_decoder(g, to):
    """rows_of gives what extend takes: the rows a pool holds go to another one."""
    cfg = e2b.small_config()
    weights = e2b.Weights(cfg, seed=22)
    dec = decoder(g, cfg, weights, [5, 40])
    dec.step([1, 2])
    other = paged.PagedDecoder(g, cfg, weights, 3, max_len=96, kv_type=to, **({} if to == "f32" else dict(k_scale=SCALE, v_scale=SCALE)))
    other.extend([0, 41, 0], dec.rows_of(1))
    for layer in dec.pages:
        for a, b in zip(dec.rows_of(1)(layer), other.rows_of(1)(layer)):
            if to == "f32":
                assert np.array_equal(a.cpu().numpy(), b.cpu().numpy())
            elif to == "e2m1":
                # a block's largest code is 6 (its size over the scale is 5.6 to 6.4): the same scale again
                assert np.array_equal(a.cpu().numpy(), b.cpu().numpy())
            else:
                x = a / SCALE
                assert np.array_equal((x.clamp(-448, 448).to(b.new_empty(0).to(g._torch.float8_e4m3fn).dtype).float() * SCALE).cpu().numpy(),
                                      b.cpu().numpy())
    for bad in (-1, 2):
        with pytest.raises(GqError):
            dec.rows_of(bad)
    dec.close()
    other.close()


def test_options_of_each_request(g):
    """Every place draws with its own options from its own state; idle places draw nothing."""
    torch = g._torch
    cfg = e2b.small_config()
    weights = e2b.Weights(cfg, seed=23)
    lens = [4, 9, 0, 30, 12]
    dec = decoder(g, cfg, weights, lens, sample=None, seed=77)
    dec.end([2])
    f32 = lambda *a: torch.tensor(a, device=g.torch_device)  # noqa: E731
    t, k, p, low = [1.0, 0.0, 1.0, 0.7, 1.4], [0, 5, 0, 8, 0], [1.0, 1.0, 1.0, 0.9, 0.8], [0.0, 0.0, 0.0, 0.0, 0.05]
    dec.temperature.copy_(f32(*t))
    dec.top_p.copy_(f32(*p))
    dec.min_p.copy_(f32(*low))
    dec.top_k.copy_(f32(*k).to(torch.int32))
    state = list(range(77, 82))
    for i in range(5):
        if i == 2:
            dec.record_steps()
        dec.step([1, 2, 3, 4, 5] if i == 0 else None)
        g.flush()
        took = dec.took.tolist()
        logits, tokens, probs = dec.controlled.cpu().numpy(), dec.tokens.tolist(), dec.probs.tolist()
        for b in range(5):
            if not took[b]:
                continue
            after, u = splitmix(state[b])
            if t[b] > 0:
                state[b] = after
            want, prob, _ = sample_ref(logits[b], t[b], k[b], p[b], low[b], u)
            assert tokens[b] == want and abs(probs[b] - prob) <= 2.0 ** -22 * prob
        assert (dec.rng.cpu().numpy().view(np.uint64) == np.array(state, np.uint64))[np.array(took)].all()
        assert took == ([True] * 5 if i == 0 else [True, True, False, True, True])
    dec.close()


def test_refusals(g):
    cfg = e2b.small_config()
    cfg.head_dim = 24
    with pytest.raises(GqError) as e:
        paged.PagedDecoder(g, cfg, e2b.Weights(cfg), 1, 16, kv_type="e2m1")
    assert e.value.status == _abi.GQ_ERR_UNSUPPORTED
