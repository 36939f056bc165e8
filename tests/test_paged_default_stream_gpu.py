"""PagedDecoder over a backend on torch's default stream (needs a B200): the same steps as over one with a stream of
its own."""
import numpy as np
import pytest

from gq import CudaBackend, e2b, paged
from test_paged_decode_gpu import rows_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("sample", [(0.0, 0, 1.0), (1.0, 20, 0.9), None])
def test_steps_on_the_default_stream(sample):
    cfg = e2b.small_config()
    lens, seen = [4, 0, 30], []
    for own in (False, True):
        g = CudaBackend(0, own_stream=own)
        weights = e2b.Weights(cfg, seed=31)
        dec = paged.PagedDecoder(g, cfg, weights, len(lens), max_len=64, sample=sample, seed=5)
        dec.extend(lens, rows_of(g, cfg, weights, lens))
        got = []
        for i in range(4):
            dec.step([1, 2, 3] if i == 0 else None)
            g.flush()
            got.append((dec.tokens.tolist(), dec.rng.tolist(), dec.read(dec.logits)))
        dec.end([1])
        dec.step()
        dec.step()
        g.flush()
        got.append((dec.tokens.tolist(), dec.took.tolist(), np.array(dec.kv_bytes())))
        seen.append(got)
        dec.close()
        g.close()
    for a, b in zip(*seen):
        assert a[0] == b[0] and a[1] == b[1] and np.array_equal(a[2], b[2])
