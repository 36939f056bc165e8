"""What gq.paged.PagedDecoder keeps of its requests while others join, end and stand
still (needs a B200). The tests keep each request's ids themselves; the step's
controlled logits must equal the definition applied to its raw logits, operation by
operation in f32 (every one rounds once on both sides). Logits of two decoders of the
same step agree to relative L2 1e-4, the bound of the whole-step tests."""
import numpy as np
import pytest

from gq import CudaBackend, GqError, _abi, e2b, paged
from numerics import rel_l2

pytestmark = pytest.mark.gpu

STEP_REL = 1e-4


@pytest.fixture(scope="module")
def g():
    be = CudaBackend(0, own_stream=True)
    yield be
    be.close()


CFG = e2b.small_config()


def seeded_rows(g, lens, seed=5):
    """Keys and values of `lens` new tokens of each request, ~N(0, 1)."""
    def rows(layer):
        gen = g._torch.Generator(device=g.torch_device).manual_seed(seed + layer)
        d = CFG.heads_kv * CFG.dh(layer)
        return [g._torch.randn(sum(lens), d, generator=gen, device=g.torch_device) for _ in range(2)]
    return rows


def make(g, batch, max_len=64, seed=12, **kw):
    return paged.PagedDecoder(g, CFG, e2b.Weights(CFG, seed=seed), batch, max_len=max_len, kv_type="f32", **kw)


def set_penalties(g, dec, rep, presence, frequency):
    dec.penalties.copy_(g._torch.tensor([[rep, presence, frequency]], device=g.torch_device).expand(dec.batch, 3))
    g._torch.cuda.synchronize()


def controlled(raw, prompt, made, rep, presence, frequency):
    """The penalties' definition: ids of the prompt (None: not known) and the ids decoded since."""
    f, y = np.float32, np.array(raw, dtype=np.float32)
    for c in {t for t in list(prompt) + list(made) if t is not None}:
        y[c] = y[c] / f(rep) if y[c] > 0 else y[c] * f(rep)
        n = list(made).count(c)
        if n:
            y[c] = (y[c] - f(frequency) * f(n)) - f(presence)
    return y


PENALTIES = (1.25, 0.75, 0.5)


def check_controlled(dec, prompts, made, places):
    raw, got = dec.read(dec.logits), dec.read(dec.controlled)
    for b in places:
        np.testing.assert_array_equal(got[b], controlled(raw[b], prompts[b], made[b], *PENALTIES), err_msg=f"request {b}")


def test_a_request_that_joins_leaves_the_others_penalties_alone(g):
    """What running requests have generated stays generated: their presence and frequency
    penalties count it after another request joins."""
    dec = make(g, 3)
    set_penalties(g, dec, *PENALTIES)
    prompts, made = [[1, 2, 3], [7] * 20, []], [[], [], []]
    dec.extend([3, 20, 0], seeded_rows(g, [3, 20]), tokens=[prompts[0], prompts[1], []])
    for ids in ([5, 9, 11], [5, 7, 12], [6, 8, 12]):
        dec.step(ids)
        g.flush()
        for b in range(3):
            made[b].append(ids[b])
        check_controlled(dec, prompts, made, range(3))
    dec.end([2])
    dec.step([6, 6, 6])
    g.flush()
    prompts[2], made[2] = [30, 31, 32, 33, 34], []
    for b in (0, 1):
        made[b].append(6)
    dec.extend([0, 0, 5], seeded_rows(g, [5], seed=9), tokens=[[], [], prompts[2]])
    assert dec.prompt_lens.tolist() == [3, 20, 5]
    dec.step([5, 7, 30])
    g.flush()
    for b, t in enumerate([5, 7, 30]):
        made[b].append(t)
    check_controlled(dec, prompts, made, range(3))
    dec.close()


def test_a_prompt_without_ids_is_not_penalised(g):
    """A prompt whose ids are not given counts as no id: not as zeros, and not as what the
    place's former request said."""
    dec = make(g, 2)
    set_penalties(g, dec, *PENALTIES)
    dec.extend([4, 20], seeded_rows(g, [4, 20]), tokens=[[1, 2, 3, 4], list(range(40, 60))])
    dec.step([5, 60])
    g.flush()
    dec.end([1])
    dec.step([6, 61])
    g.flush()
    dec.extend([0, 12], seeded_rows(g, [12], seed=9))
    dec.step([7, 8])
    g.flush()
    check_controlled(dec, [[1, 2, 3, 4], []], [[5, 6, 7], [8]], range(2))
    # ids of a part of the prompt: the rest is not known
    dec.extend([0, 6], seeded_rows(g, [6], seed=10), tokens=[[], [21, 22]])
    dec.step([8, 9])
    g.flush()
    check_controlled(dec, [[1, 2, 3, 4], [8, 21, 22]], [[5, 6, 7, 8], [9]], range(2))
    dec.close()


def hold(g, dec, ms=60):
    """Keep the backend's stream busy for some milliseconds, so that what is enqueued next
    is still to come when the host goes on."""
    with g._torch.cuda.stream(dec._stream()):
        g._torch.cuda._sleep(int(ms * 1.9e6))


def test_extend_sees_the_steps_still_in_flight(g):
    """A request takes the place of one that ended in a step not yet done: its ids go to the
    start of the place's history."""
    dec = make(g, 2)
    set_penalties(g, dec, *PENALTIES)
    dec.extend([4, 20], seeded_rows(g, [4, 20]), tokens=[[1, 2, 3, 4], list(range(40, 60))])
    dec.step([5, 60])  # (a first step allocates, which waits for the device)
    g.flush()
    dec.tokens.copy_(g._torch.tensor([6, 61], device=g.torch_device))
    dec.end([1])
    hold(g, dec)
    dec.step()  # (ids from the host would wait for the stream)
    dec.extend([0, 3], seeded_rows(g, [3], seed=9), tokens=[[], [30, 31, 32]])
    assert dec.lens.tolist() == [6, 3]
    assert dec.history[1, :3].tolist() == [30, 31, 32]
    dec.tokens.copy_(g._torch.tensor([7, 33], device=g.torch_device))
    g._torch.cuda.synchronize()
    hold(g, dec)
    dec.step()
    size = 2 * CFG.heads_kv * 4
    want = sum(size * CFG.dh(i) * min(n, CFG.window_of(i) or n) for n in (7, 4) for i in range(CFG.layers))
    assert dec.kv_bytes() == want
    g.flush()
    check_controlled(dec, [[1, 2, 3, 4], [30, 31, 32]], [[5, 6, 7], [33]], range(2))
    dec.close()


def test_an_earlier_steps_error_takes_nothing(g):
    """An error that a step left behind is raised before extend takes pages: its rows are
    not left out of pages that it took."""
    dec = make(g, 2, n_pages=3)
    dec.extend([32, 0], seeded_rows(g, [32]))
    dec.step([1, 2])  # one page is left, two are needed
    with pytest.raises(GqError) as e:
        dec.extend([0, 5], seeded_rows(g, [5], seed=9))
    assert e.value.status == _abi.GQ_ERR_DEVICE
    assert dec.lens.tolist() == [32, 0] and int(dec.count[0]) == 1
    rows = seeded_rows(g, [5], seed=9)
    dec.extend([0, 5], rows)
    assert dec.lens.tolist() == [32, 5] and int(dec.count[0]) == 0
    for layer, pages in dec.pages.items():
        k, v = rows(layer)
        at = dec.table[1, 0].long()
        assert g._torch.equal(pages.k[at, 0, :5], k) and g._torch.equal(pages.v[at, 0, :5], v)
    dec.close()


def alone(g, rows, ids):
    """Logits of decoding `ids` after the cache `rows` of one request, in a decoder of its own."""
    dec = make(g, 1)
    n = rows(0)[0].shape[0]
    dec.extend([n], rows)
    for t in ids:
        dec.step([t])
    g.flush()
    out = dec.read(dec.logits)[0].copy()
    dec.close()
    return out


def test_a_request_that_takes_an_ended_place_at_once(g):
    """end, then extend with no step between: the place begins anew, and the former
    request's pages are back."""
    dec = make(g, 2, n_pages=4)
    dec.extend([40, 3], seeded_rows(g, [40, 3]), tokens=[[9] * 40, [1, 2, 3]])
    assert int(dec.count[0]) == 0
    dec.end([0])
    rows = seeded_rows(g, [18], seed=9)
    dec.extend([18, 0], rows, tokens=[[5] * 18, []])
    assert dec.lens.tolist() == [18, 3] and int(dec.count[0]) == 1
    assert dec.history[0, :18].tolist() == [5] * 18
    dec.step([7, 8])
    g.flush()
    assert dec.lens.tolist() == [19, 4] and dec.prompt_lens.tolist() == [18, 3]
    assert rel_l2(dec.read(dec.logits)[0], alone(g, rows, [7])) <= STEP_REL
    # a place that ended and is not extended still waits for its step
    dec.end([1])
    dec.extend([2, 0], seeded_rows(g, [2], seed=11))
    assert dec.lens.tolist() == [21, 4]
    dec.step([7, 8])
    g.flush()
    assert dec.lens.tolist() == [22, 0]
    dec.close()


def test_controls_and_tokens_follow_the_callers_stream(g):
    """What torch's current stream does before a step is in it, what it does after comes
    after it, and it sees the step's tokens and lengths, all without a synchronisation."""
    torch = g._torch
    dec = make(g, 2)
    dec.extend([3, 4], seeded_rows(g, [3, 4]), tokens=[[1, 2, 3], [4, 5, 6, 7]])
    new = torch.tensor([PENALTIES] * 2, device=g.torch_device)
    prompts, made, tokens = [[1, 2, 3], [4, 5, 6, 7]], [[], []], [8, 9]
    dec.tokens.copy_(torch.tensor(tokens, device=g.torch_device))
    for record in (False, True):
        if record:
            dec.record_steps()
        dec.penalties.copy_(torch.tensor([[1.0, 0.0, 0.0]] * 2, device=g.torch_device))
        torch.cuda.synchronize()
        torch.cuda._sleep(100_000_000)  # the change below is still to come when step returns
        dec.penalties.copy_(new)
        dec.step()
        for b in range(2):
            made[b].append(tokens[b])
        tokens = dec.tokens.tolist()
        g.flush()
        check_controlled(dec, prompts, made, range(2))
        hold(g, dec)
        dec.step()
        dec.penalties.fill_(2.0)  # the step, still in flight, does not see it
        for b in range(2):
            made[b].append(tokens[b])
        tokens = dec.tokens.tolist()
        assert dec.lens.tolist() == [3 + len(made[0]), 4 + len(made[1])]
        g.flush()
        check_controlled(dec, prompts, made, range(2))
        assert tokens == np.argmax(dec.read(dec.controlled), 1).tolist()
    # a change on another stream of the caller's
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        torch.cuda._sleep(100_000_000)
        dec.penalties.copy_(new)
        dec.step()
    for b in range(2):
        made[b].append(tokens[b])
    g.flush()
    check_controlled(dec, prompts, made, range(2))
    dec.close()


@pytest.mark.parametrize("recorded", [False, True])
def test_a_refused_step_can_be_repeated(g, recorded):
    """Too few pages for a step: tokens, random states, lengths and pages are as before, and
    the next step that fits goes on from there."""
    dec = make(g, 2, n_pages=4, sample=(1.0, 8, 0.95))
    rows = seeded_rows(g, [31])
    dec.extend([31, 0], rows)
    dec.extend([0, 15], seeded_rows(g, [15], seed=9))
    if recorded:
        dec.record_steps()
    assert dec.took.tolist() == [False, False]
    dec.step([5, 6])
    g.flush()
    state = lambda: [t.tolist() for t in (dec.tokens, dec.rng, dec.lens, dec.count)]  # noqa: E731
    before = state()
    assert before[2] == [32, 16] and before[3] == [1] and dec.took.tolist() == [True, True]
    for _ in range(2):  # two pages are needed
        dec.step()
        with pytest.raises(GqError) as e:
            g.flush()
        assert e.value.status == _abi.GQ_ERR_DEVICE
        assert state() == before and dec.took.tolist() == [False, False]
    if not recorded:
        with pytest.raises(GqError):
            dec.record_steps()
        assert state() == before
    dec.end([1])
    dec.step()  # refused too, and gives the ended request's page back
    with pytest.raises(GqError):
        g.flush()
    assert state() == [before[0], before[1], [32, 0], [2]]
    dec.step()
    g.flush()
    assert dec.lens.tolist()[0] == 33 and dec.took.tolist()[0]
    assert dec.history[0, 31:33].tolist() == [5, before[0][0]]
    assert rel_l2(dec.read(dec.logits)[0], alone(g, rows, [5, before[0][0]])) <= STEP_REL
    dec.close()


@pytest.mark.parametrize("recorded", [False, True])
def test_places_without_a_token_take_no_page(g, recorded):
    """In a full pool an idle place and a request at max_len do not stop the others, whose
    rows go to their own places; the idle ones' tokens and random states stay."""
    lens = [5, 47, 31, 17]
    dec = make(g, 4, max_len=48, n_pages=8, sample=(1.0, 8, 0.95))
    rows = [seeded_rows(g, [n], seed=20 + n) for n in lens]
    for b, n in enumerate(lens):
        dec.extend([n if i == b else 0 for i in range(4)], rows[b])
    assert int(dec.count[0]) == 0
    if recorded:
        dec.record_steps()
    dec.end([0])
    dec.step([1, 2, 3, 4])
    g.flush()
    assert dec.lens.tolist() == [0, 48, 32, 18] and dec.took.tolist() == [True] * 4 and int(dec.count[0]) == 1
    said, tokens, states = [[3], [4]], dec.tokens.tolist(), dec.rng.tolist()
    for i in range(10):  # the first takes the last page
        dec.step()
        g.flush()
        assert dec.lens.tolist() == [0, 48, 33 + i, 19 + i] and dec.took.tolist() == [False, False, True, True]
        for k, b in enumerate((2, 3)):
            said[k].append(tokens[b])
        now = dec.tokens.tolist()
        assert now[:2] == tokens[:2] and dec.rng.tolist()[:2] == states[:2]
        tokens = now
    assert int(dec.count[0]) == 0
    logits = dec.read(dec.logits)
    for k, b in enumerate((2, 3)):
        assert rel_l2(logits[b], alone(g, rows[b], said[k])) <= STEP_REL
    dec.end([1])
    dec.step()  # (a full request has no last step to take)
    g.flush()
    assert dec.lens.tolist() == [0, 0, 43, 29] and int(dec.count[0]) == 3
    dec.extend([17, 0, 0, 0], seeded_rows(g, [17], seed=60))
    dec.step()
    g.flush()
    assert dec.lens.tolist() == [18, 0, 44, 30] and dec.took.tolist() == [True, False, True, True]
    dec.close()


def test_no_request_passes_max_len(g):
    """max_len is the limit where the last page could hold more, in steps and in extend; the
    ids of a request that stands still there are not written over."""
    dec = make(g, 2, max_len=20)  # pages of 16
    set_penalties(g, dec, *PENALTIES)
    prompt, said = list(range(40, 58)), [[60, 61], [1, 2]]
    dec.extend([18, 0], seeded_rows(g, [18]), tokens=[prompt, []])
    for ids in zip(*said):
        dec.step(list(ids))
    for i in range(3):
        dec.step([70 + i, 3 + i])
        said[1].append(3 + i)
    g.flush()
    assert dec.lens.tolist() == [20, 5] and dec.history[0].tolist() == prompt + said[0]
    check_controlled(dec, [prompt, []], said, range(2))
    for lens, tokens in (([1, 0], None), ([0, 16], None), ([0], None), ([0, 0, 0], None), ([0, -1], None),
                         ([0, 2], [[], [1, 2, 3]]), ([0, 0], [[], [], []])):
        with pytest.raises(GqError) as e:
            dec.extend(lens, seeded_rows(g, [sum(lens)]), tokens=tokens)
        assert e.value.status == _abi.GQ_ERR_INVALID_ARGUMENT
    assert dec.lens.tolist() == [20, 5]
    dec.extend([0, 15], seeded_rows(g, [15], seed=8))
    assert dec.lens.tolist() == [20, 20]
    dec.end([0])
    dec.extend([20, 0], seeded_rows(g, [20], seed=8))  # the ended request's tokens do not count
    assert dec.lens.tolist() == [20, 20]
    dec.close()


def test_biases_and_masks_of_a_decoder_are_checked(g):
    """Too short for the batch, of another type or on the host: refused when the decoder is
    made, not read past when it steps."""
    torch, dev = g._torch, g.torch_device
    i32 = lambda *a: torch.tensor(a, dtype=torch.int32, device=dev)  # noqa: E731
    ids, values, offsets = i32(5, 6), torch.tensor([30.0, 1.0], device=dev), i32(0, 1, 2)
    words, rows = torch.full((2, CFG.vocab // 32), -1, dtype=torch.int32, device=dev), i32(0, 1)
    for kw in (dict(bias=(ids, values, offsets[:2])), dict(bias=(ids, values[:1], offsets)), dict(bias=(ids.long(), values, offsets)),
               dict(bias=(ids, values, offsets.cpu())), dict(masks=(words, rows[:1])), dict(masks=(words[:, 1:], rows)),
               dict(masks=(words[:1], None)), dict(masks=(words[:, :-1].contiguous(), rows)), dict(masks=(words[0], rows))):
        with pytest.raises(GqError) as e:
            make(g, 2, **kw)
        assert e.value.status == _abi.GQ_ERR_INVALID_ARGUMENT
    dec = make(g, 2, bias=(ids, 1000 * values, offsets), masks=(words, rows))
    assert dec.step([1, 1]).tolist() == [5, 6]
    g.flush()
    dec.close()


def test_a_refused_extend_of_an_ended_place_leaves_it_idle(g):
    """The ended request's pages have gone back; the place takes none of them until a request
    has it."""
    dec = make(g, 2, n_pages=4)
    dec.extend([20, 31], seeded_rows(g, [20, 31]))
    dec.end([0])
    with pytest.raises(GqError):
        dec.extend([48, 0], seeded_rows(g, [48]))  # three pages, two are back
    assert dec.lens.tolist() == [0, 31] and int(dec.count[0]) == 2
    for n in (32, 33):
        dec.step([1, 2])
        g.flush()
        assert dec.lens.tolist() == [0, n] and dec.took.tolist() == [False, True]
    dec.extend([5, 0], seeded_rows(g, [5]))
    dec.step([1, 2])
    g.flush()
    assert dec.lens.tolist() == [6, 34] and dec.took.tolist() == [True, True]
    dec.close()


def test_places_that_are_not_there_cannot_end(g):
    dec = make(g, 2)
    dec.extend([3, 4], seeded_rows(g, [3, 4]))
    for places in ([2], [-1], [0, 5]):
        with pytest.raises(GqError) as e:
            dec.end(places)
        assert e.value.status == _abi.GQ_ERR_INVALID_ARGUMENT
    dec.end([])
    dec.step([1, 2])
    g.flush()
    assert dec.lens.tolist() == [4, 5]
    dec.close()
