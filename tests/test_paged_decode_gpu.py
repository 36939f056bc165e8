"""The decode step over pages (gq.paged.PagedDecoder) against the contiguous decoder,
request by request (needs a B200): the same weights and cache contents, f32 pages, so
both compute the same step; relative L2 of the logits at most 1e-4, the bound of the
whole-step tests."""
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


def contiguous(g, cfg, weights, length, ids):
    """Logits of the steps `ids` of one sequence whose cache holds `length` seeded tokens."""
    dec = e2b.Decoder(g, cfg, weights, 1, length, capacity=length + len(ids) + 1)
    out = []
    for i, t in enumerate(ids):
        dec.set_position(length + i)
        dec.set_ids([t])
        dec.run()
        out.append(dec.read(dec.logits)[0].copy())
    dec.close()
    return out


def rows_of(g, cfg, weights, lens):
    """The seeded caches of the contiguous decoders, in request order."""
    def rows(layer):
        d = cfg.heads_kv * cfg.dh(layer)
        kv = [weights.kv_prefix(layer, 1, n) for n in lens if n]
        return [g._torch.from_numpy(np.concatenate([np.asarray(p[j]).reshape(-1, d) for p in kv]).astype(np.float32)).to(g.torch_device)
                for j in range(2)]
    return rows


@pytest.mark.parametrize("make,page_size", [(e2b.small_config, 16), (e2b.tiny_config, 4)])
def test_steps_match_the_contiguous_decoder(g, make, page_size):
    cfg = make()
    weights = e2b.Weights(cfg, seed=11)
    lens = [0, 1, 15, 16, 33, 70]
    steps = np.random.default_rng(3).integers(0, cfg.vocab, (4, len(lens)))
    dec = paged.PagedDecoder(g, cfg, weights, len(lens), max_len=80, page_size=page_size, kv_type="f32")
    dec.extend(lens, rows_of(g, cfg, weights, lens))
    want = [contiguous(g, cfg, weights, n, steps[:, b]) for b, n in enumerate(lens)]
    for i, ids in enumerate(steps):
        if i == 2:
            dec.record_steps()  # the rest from a graph
        dec.step(ids)
        g.flush()
        logits = dec.read(dec.logits)
        tokens = dec.tokens.cpu().numpy()
        for b in range(len(lens)):
            assert rel_l2(logits[b], want[b][i]) <= STEP_REL, (i, b)
            assert tokens[b] == np.argmax(logits[b])  # greedy, no penalty
    assert dec.lens.tolist() == [n + 4 for n in lens]
    used = sum(-(-(n + 4) // page_size) for n in lens)
    assert int(dec.count[0]) == dec.n_pages - used
    dec.close()


def test_requests_end_and_others_begin(g):
    cfg = e2b.small_config()
    weights = e2b.Weights(cfg, seed=12)
    lens = [40, 7, 25]
    dec = paged.PagedDecoder(g, cfg, weights, 3, max_len=64, kv_type="f32", n_pages=9)
    dec.extend(lens, rows_of(g, cfg, weights, lens))
    dec.step([1, 2, 3])
    g.flush()
    dec.end([0])
    dec.step([4, 5, 6])  # the last of request 0, whose pages go back after it
    g.flush()
    assert dec.lens.tolist() == [0, 9, 27]
    assert int(dec.count[0]) == 9 - 1 - 2
    dec.step([0, 7, 8])  # place 0 idles
    g.flush()
    assert dec.lens.tolist() == [0, 10, 28]
    dec.extend([33, 0, 0], rows_of(g, cfg, weights, [33]))
    dec.step([9, 10, 11])
    g.flush()
    assert dec.lens.tolist() == [34, 11, 29]
    assert rel_l2(dec.read(dec.logits)[0], contiguous(g, cfg, weights, 33, [9])[0]) <= STEP_REL
    # more than the pool holds: refused as a whole, and nothing is lost
    with pytest.raises(GqError) as e:
        dec.extend([29, 40, 0], rows_of(g, cfg, weights, [29, 40]))
    assert e.value.status == _abi.GQ_ERR_DEVICE
    assert dec.lens.tolist() == [34, 11, 29] and int(dec.count[0]) == 9 - 3 - 1 - 2
    dec.step([12, 13, 14])
    g.flush()
    assert dec.lens.tolist() == [35, 12, 30]
    dec.close()


@pytest.mark.parametrize("kv_type", ["f16", "bf16", "e4m3"])
def test_controls_and_narrow_pages(g, kv_type):
    """The pages hold the prompts' rows rounded to their type; masks and penalties steer the
    tokens."""
    torch = g._torch
    cfg = e2b.small_config()
    weights = e2b.Weights(cfg, seed=13)
    lens, V = [50, 3], cfg.vocab
    words = torch.zeros(1, V // 32, dtype=torch.int32, device=g.torch_device)
    words[0, 3] = 0b1010  # request 0 may say 97 or 99
    rows = torch.tensor([0, -1], dtype=torch.int32, device=g.torch_device)
    scale = 1 / 16 if kv_type == "e4m3" else 1.0
    dec = paged.PagedDecoder(g, cfg, weights, 2, max_len=64, kv_type=kv_type, k_scale=scale, v_scale=scale, masks=(words, rows))
    dec.extend(lens, rows_of(g, cfg, weights, lens), tokens=[[5] * 50, [6, 7, 8]])
    for layer, pages in dec.pages.items():
        for pool, rows_l in zip((pages.k, pages.v), rows_of(g, cfg, weights, lens)(layer)):
            at = torch.arange(50, device=g.torch_device)
            got = pool[dec.table[0].long()[at // 16], :, at % 16].float()
            x = rows_l[:50].view(got.shape)
            assert torch.equal(got, ((x / scale).clamp(-448, 448) if kv_type == "e4m3" else x).to(pool.dtype).float())
    dec.step([1, 1])
    g.flush()
    logits = dec.read(dec.logits)
    first = dec.tokens.tolist()
    assert first[0] in (97, 99) and first[1] == int(np.argmax(logits[1]))
    # what was said (and the prompt's ids) becomes impossible under a large penalty
    dec.penalties.copy_(torch.tensor([[1.0, 1e6, 0.0]], device=g.torch_device))
    dec.step()
    g.flush()
    second = dec.tokens.tolist()
    assert second[0] in (97, 99) and second[0] != first[0]
    assert second[1] not in (1, first[1])
    assert dec.history[1, :5].tolist() == [6, 7, 8, 1, first[1]]
    dec.close()


def test_refusals(g):
    with pytest.raises(GqError) as e:
        paged.PagedDecoder(g, e2b.tiny_config(), e2b.Weights(e2b.tiny_config()), 1, 16, kv_type="int4")
    assert e.value.status == _abi.GQ_ERR_UNSUPPORTED
