"""PagedDecoder's `probs` (needs a B200): the probabilities that the places' tokens were drawn with, also after the step
was recorded, and of places that a step took no token of."""
import pytest

from gq import CudaBackend, GqError, e2b, paged
from test_paged_decode_gpu import rows_of

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def g():
    be = CudaBackend(0, own_stream=True)
    yield be
    be.close()


def decoder(g, lens, **kw):
    cfg = e2b.small_config()
    weights = e2b.Weights(cfg, seed=41)
    dec = paged.PagedDecoder(g, cfg, weights, len(lens), max_len=64, sample=None, seed=9, **kw)
    dec.extend(lens, rows_of(g, cfg, weights, lens))
    return dec


def test_recording_leaves_the_probabilities(g):
    dec = decoder(g, [4, 9])
    dec.step([1, 2])
    g.flush()
    tokens, probs = dec.tokens.tolist(), dec.probs.tolist()
    assert all(0 < p < 1 for p in probs)
    dec.record_steps()
    assert dec.tokens.tolist() == tokens and dec.probs.tolist() == probs
    dec.step()
    g.flush()
    assert dec.probs.tolist() != probs
    dec.close()


def test_idle_places_keep_theirs(g):
    dec = decoder(g, [4, 9, 62])
    dec.step([1, 2, 3])
    dec.end([1])
    dec.step()
    g.flush()
    tokens, probs = dec.tokens.tolist(), dec.probs.tolist()
    for _ in range(2):  # place 1 idles, and 2 stands still at max_len
        dec.step()
        g.flush()
        assert dec.took.tolist() == [True, False, False]
        assert dec.tokens.tolist()[1:] == tokens[1:] and dec.probs.tolist()[1:] == probs[1:]
    dec.close()


def test_a_step_without_pages_keeps_them(g):
    dec = decoder(g, [16, 15], n_pages=3)
    dec.step([1, 2])  # the last page
    g.flush()
    tokens, probs = dec.tokens.tolist(), dec.probs.tolist()
    dec.step()  # place 1 wants one more
    with pytest.raises(GqError):
        g.flush()
    assert dec.tokens.tolist() == tokens and dec.probs.tolist() == probs
    dec.close()


def test_a_request_that_nothing_is_left_of(g):
    """Token -1 with probability 0; it goes on with another id."""
    torch = g._torch
    words = torch.full((2, -(-e2b.small_config().vocab // 32)), -1, dtype=torch.int32, device=g.torch_device)
    words[1] = 0
    rows = torch.tensor([0, 1], dtype=torch.int32, device=g.torch_device)
    dec = decoder(g, [4, 9], masks=(words, rows))
    dec.step([1, 2])
    g.flush()
    assert dec.tokens[1] == -1 and dec.probs[1] == 0 and dec.tokens[0] >= 0 and dec.probs[0] > 0
    dec.tokens[1] = 5
    rows[1] = 0
    dec.step()
    g.flush()
    assert dec.lens.tolist() == [6, 11] and dec.tokens.min() >= 0 and dec.probs.min() > 0
    rows[1] = 1
    dec.step()
    g.flush()
    assert dec.tokens[1] == -1
    dec.step()
    with pytest.raises(GqError):
        g.flush()
    dec.close()
