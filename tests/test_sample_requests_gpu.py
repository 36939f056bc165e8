"""A token for each request with options of its own (gq_sample_requests) against the definition in 64
bits (needs a B200). Tokens must be equal: the kernel's running sums are off by less than 1e-10 of
the whole, so a random number next to the border of two tokens would have to be that close to it.
Probabilities: within 2^-23 (one f32 rounding, of a quotient that is exact to 2^-40), or within
2^-40 of the row's largest weight, what its multiples of 2^-44 leave to a small one."""
import ctypes

import numpy as np
import pytest

from gq import CudaBackend, GqError, _abi

pytestmark = pytest.mark.gpu

PROB_REL, PROB_ABS = 2.0 ** -23, 2.0 ** -40


@pytest.fixture(scope="module")
def g():
    be = CudaBackend(0)
    yield be
    be.close()


def dev(g, a, dtype=None):
    return g._torch.from_numpy(np.ascontiguousarray(a, dtype=dtype)).to(g.torch_device)


def sample_ref(row, t, k, p, low, u):
    """Token and probability of one row, and how many tokens the options leave."""
    row = np.where(np.isnan(row), -np.inf, row.astype(np.float64))
    top = row.max()
    if top == -np.inf:
        return -1, 0.0, 0
    if not t > 0:
        return int(np.argmax(row)), 1.0, 1
    with np.errstate(invalid="ignore", over="ignore"):
        w = np.where(row == top, 1.0, np.where(row == -np.inf, 0.0, np.exp((row - top) / np.float64(np.float32(t)))))
    w = np.nan_to_num(w, nan=0.0)
    order = np.argsort(-row, kind="stable")
    s = w[order]
    n = min(len(s), int(k)) if k > 0 else len(s)
    p = np.float64(np.float32(p))
    if p < 1:
        run = np.cumsum(s[:n])
        n = min(n, int((run < p * run[-1]).sum()) + 1)
    n = max(1, min(n, int((s >= min(max(np.float64(np.float32(low)), 0.0), 1.0)).sum())))
    n = min(n, int((s > 0).sum()))
    left = np.zeros_like(w)
    left[order[:n]] = s[:n]
    run = np.cumsum(left)
    u = min(max(u, 0.0), 1 - 2.0 ** -53) if u == u else 0.0
    at = min(int((run <= u * run[-1]).sum()), int(np.flatnonzero(left)[-1]))
    return at, left[at] / run[-1], n


def check(g, logits, t=None, k=None, p=None, low=None, u=None, ld=None):
    torch = g._torch
    m, v = logits.shape
    if ld:
        store = torch.full((m, ld), 99.0, device=g.torch_device)
        store[:, :v] = dev(g, logits, np.float32)
        x = store[:, :v]
    else:
        x = dev(g, logits, np.float32)
    probs = torch.full((m,), -5.0, device=g.torch_device)
    kw = {n: dev(g, a, dt) for n, a, dt in (("temperature", t, np.float32), ("top_k", k, np.int32), ("top_p", p, np.float32),
                                             ("min_p", low, np.float32), ("uniforms", u, np.float64)) if a is not None}
    tokens = g.sample_requests(x, probs=probs, **kw).cpu().numpy()
    probs = probs.cpu().numpy()
    left = []
    for i in range(m):
        want, prob, n = sample_ref(logits[i].astype(np.float32), 1.0 if t is None else np.float32(t[i]), 0 if k is None else k[i],
                                   1.0 if p is None else p[i], 0.0 if low is None else low[i], u[i])
        assert tokens[i] == want, (i, tokens[i], want, n)
        assert abs(probs[i] - prob) <= PROB_REL * prob + PROB_ABS, (i, probs[i], prob)
        left.append(n)
    return tokens, left


def options(rng, m):
    t = np.where(rng.random(m) < 0.15, 0.0, rng.uniform(0.3, 1.6, m)).astype(np.float32)
    k = rng.choice([0, 0, 1, 2, 20, 64, 1000, 10 ** 9], m).astype(np.int32)
    p = rng.choice([1.0, 1.5, 0.95, 0.5, 0.01, 0.999], m).astype(np.float32)
    low = rng.choice([0.0, 0.0, -1.0, 0.05, 0.001, 1.0], m).astype(np.float32)
    return t, k, p, low, rng.random(m)


@pytest.mark.parametrize("m,v", [(1, 1), (3, 2), (5, 3), (2, 31), (40, 33), (300, 127), (64, 1000), (7, 4099), (16, 32003), (150, 32000),
                                 (20, 50257), (3, 131071), (1, 262144), (9, 262144), (33, 262144), (2, 300007), (1, 524288), (4, 524287)])
def test_tokens_match_the_definition(g, m, v):
    rng = np.random.default_rng(m * 1000003 + v)
    x = 2.5 * rng.standard_normal((m, v)).astype(np.float32)
    for i in range(m):
        x[i, rng.integers(0, v, 20)] += rng.uniform(0, 14, 20).astype(np.float32)
    t, k, p, low, u = options(rng, m)
    check(g, x, t, k, p, low, u)
    check(g, x, u=u)  # every option off
    check(g, x, t=t, p=np.full(m, 0.9, np.float32), u=u, ld=v + 5)


@pytest.mark.parametrize("v", [7, 5000, 262144])
def test_equal_logits(g, v):
    """Ties go to the smaller id: of a row of one number the options leave its first tokens."""
    rng = np.random.default_rng(v)
    m = 24
    x = np.full((m, v), -3.25, np.float32)
    x[8:16] = rng.choice([0.0, -0.0, 1.0], (8, v)).astype(np.float32)  # two values, zeros of both signs
    x[16:] = np.round(rng.standard_normal((8, v)) * 3) / 3
    k = np.array([1, 3, v // 2, 0, 0, 0, v, v - 1] * 3, np.int32)
    p = np.array([1, 1, 1, 0.25, 0.75, 0.5, 0.5, 1] * 3, np.float32)
    for u in (np.zeros(m), np.full(m, 1 - 2.0 ** -53), rng.random(m)):
        _, left = check(g, x, k=k, p=p, u=u)
    assert left[:4] == [1, 3, v // 2, -(-v // 4)]


def test_masked_and_special_rows(g):
    rng = np.random.default_rng(2)
    v = 3000
    x = rng.standard_normal((16, v)).astype(np.float32)
    x[0] = -np.inf
    x[1] = np.nan
    x[2, :] = -np.inf
    x[2, 1234] = -1e30  # one token allowed
    x[3, 5] = np.inf
    x[4, [7, 2000, 2999]] = np.inf
    x[5, ::2] = np.nan
    x[6] = np.where(rng.random(v) < 0.99, -np.inf, x[6])
    x[7] = 3.4e38 * rng.choice([-1, 1], v)
    x[8] = np.float32(1e-42) * rng.integers(0, 5, v)
    x[9, 0] = 200.0
    x[10, :] = np.nan
    x[10, 17] = -np.inf
    for t in (1.0, 0.0, -2.0, np.nan, 1e-30, 1e-45, 1e30, np.inf):
        for k, p, low in ((0, 1.0, 0.0), (5, 0.9, 0.0), (0, 0.5, 0.0), (4000, 1.0, 0.3)):
            f = lambda a, dt=np.float32: np.full(16, a, dt)  # noqa: E731
            check(g, x, f(t), f(k, np.int32), f(p), f(low), rng.random(16))


def test_borders_of_the_options(g):
    """top_p and min_p where a sum or a weight reaches them exactly, 0 and above 1; random numbers
    outside [0, 1)."""
    x = np.full((12, 64), -np.inf, np.float32)
    x[:, [3, 20, 21, 60]] = 0.0  # weights of exactly 1
    p = np.array([0.25, 0.5, 0.75, 0.0, -1.0, 1.0, 2.0, 0.2500001, 0.2499999, 0.7500001, 1e-38, 0.99999994], np.float32)
    _, left = check(g, x, p=p, u=np.full(12, 0.9))
    assert left == [1, 2, 3, 1, 1, 4, 4, 2, 1, 4, 1, 4]
    x[:, 20] = -1.0
    low = np.array([1.0, 2.0, 0.0, -1.0, 0.36, 0.37, 0.367, 0.368, 0.9, 0.3678, 1e-38, 0.5], np.float32)
    _, left = check(g, x, low=low, u=np.full(12, 0.999))
    assert left == [3, 3, 4, 4, 4, 3, 4, 3, 3, 4, 4, 3]
    check(g, x, u=np.array([0.0, -0.0, -1.0, 1.0, 2.0, np.nan, np.inf, -np.inf, 0.25, 0.5, 1e-300, 1 - 2.0 ** -53]))


def test_states_give_the_numbers(g):
    """rng_state: the draw of gq_sample_rows' generator, advanced by the rows that draw."""
    m, v = 9, 5000
    rng = np.random.default_rng(4)
    x = rng.standard_normal((m, v)).astype(np.float32)
    t = np.array([1, 0, 0.7, 1, -1, 1, 1, 0, 2], np.float32)
    state = [int(z) for z in rng.integers(0, 2 ** 64, m, dtype=np.uint64)]
    d = dev(g, np.array(state, np.uint64).view(np.int64))
    for _ in range(3):
        tokens = g.sample_requests(dev(g, x), temperature=dev(g, t), rng_state=d).cpu().numpy()
        for i in range(m):
            u = 0.0
            if t[i] > 0:
                z = state[i] = (state[i] + 0x9e3779b97f4a7c15) % 2 ** 64
                z = ((z ^ (z >> 30)) * 0xbf58476d1ce4e5b9) % 2 ** 64
                z = ((z ^ (z >> 27)) * 0x94d049bb133111eb) % 2 ** 64
                u = ((z ^ (z >> 31)) >> 11) / 2 ** 53
            assert tokens[i] == sample_ref(x[i], t[i], 0, 1.0, 0.0, u)[0]
        assert d.cpu().numpy().view(np.uint64).tolist() == state


def test_greedy_agrees_with_sample_rows(g):
    torch = g._torch
    x = torch.randn(5, 40000, device=g.torch_device)
    x[2, 100] = x[2, 39999] = x[2].max() + 1
    want, got = (torch.empty(5, dtype=torch.int32, device=g.torch_device) for _ in range(2))
    opts = _abi.SampleOpts(0.0, 0, 1.0, 1.0)
    zero = torch.zeros(5, dtype=torch.float64, device=g.torch_device)
    states = torch.zeros(5, dtype=torch.int64, device=g.torch_device)
    assert g.lib.gq_sample_rows(g.ctx, x.data_ptr(), 5, 40000, 0, ctypes.byref(opts), None, 0, 0, states.data_ptr(),
                                want.data_ptr()) == _abi.GQ_OK
    g.sample_requests(x, temperature=zero.float(), uniforms=zero, tokens=got)
    g.flush()
    assert torch.equal(want, got) and int(got[2]) == 100


def test_recorded_and_on_two_contexts():
    contexts = [CudaBackend(0, own_stream=True) for _ in range(2)]
    torch = contexts[0]._torch
    m, v = 12, 70001
    work = []
    for i, g in enumerate(contexts):
        gen = torch.Generator(device=g.torch_device)
        gen.manual_seed(i)
        s = dict(x=torch.randn(m, v, generator=gen, device=g.torch_device), u=torch.rand(m, dtype=torch.float64, generator=gen, device=g.torch_device),
                 p=torch.full((m,), 0.8, device=g.torch_device), tokens=torch.zeros(m, dtype=torch.int32, device=g.torch_device))
        torch.cuda.synchronize()
        s["graph"] = g.record(lambda g=g, s=s: g.sample_requests(s["x"], top_p=s["p"], uniforms=s["u"], tokens=s["tokens"]))
        work.append((g, s))
    for i in range(20):
        for g, s in work:
            s["u"].copy_(torch.rand(m, dtype=torch.float64))
            s["x"].mul_(1.05)
        torch.cuda.synchronize()
        if i == 3:  # (a larger call of the same contexts meanwhile)
            for g, s in work:
                g.sample_requests(torch.zeros(300, v, device=g.torch_device), uniforms=torch.zeros(300, dtype=torch.float64, device=g.torch_device))
        for g, s in work:
            g.replay(s["graph"])
        for g, s in work:
            g.flush()
            if i % 7 == 0:
                x, u = s["x"].cpu().numpy(), s["u"].cpu().numpy()
                assert s["tokens"].tolist() == [sample_ref(x[r], 1.0, 0, 0.8, 0.0, u[r])[0] for r in range(m)]
    for g, s in work:
        g.destroy_graph(s["graph"])
        g.close()


@pytest.mark.parametrize("v", [20011, 262144])
def test_borders_that_lie_far_down(g, v):
    """Options that leave more tokens than the pieces of a row give by themselves."""
    rng = np.random.default_rng(v + 1)
    m = 20
    x = rng.standard_normal((m, v)).astype(np.float32)
    x[4:8] = np.sort(x[4:8], axis=1)[:, ::-1]  # all that counts in the first columns
    x[8:12] *= 1e-3
    x[10:12, :3000] = 0.5  # many of one kind at the border, and outliers above them
    x[10:12, 5] = [9.0, 300.0]
    x[12, [3, v // 2, v - 1]] = np.inf
    x[13, rng.random(v) < 0.7] = np.inf
    x[14, ::3] = np.nan
    x[15] = np.where(rng.random(v) < 0.5, -np.inf, x[15])
    x[16:18] = rng.standard_cauchy((2, v)).astype(np.float32)
    x[18:] = rng.random((2, v)).astype(np.float32) * np.float32(1e38)
    t = np.ones(m, np.float32)
    t[18:] = 1e37
    f = lambda a, dt=np.float32: np.full(m, a, dt)  # noqa: E731
    for p in (0.3, 0.95, 0.9999999):
        check(g, x, t, p=f(p), u=rng.random(m))
    _, left = check(g, x, t, f(v // 3, np.int32), u=rng.random(m))
    assert left[0] == v // 3
    check(g, x, t, f(v // 3, np.int32), f(0.9), u=rng.random(m))
    check(g, x, t, f(5000, np.int32), f(0.99), f(1e-3), u=rng.random(m))
    check(g, x, t, p=f(0.9), low=f(0.05), u=rng.random(m))
    check(g, x, t, low=f(0.02), u=rng.random(m))
    check(g, x[:18], 30 * t[:18], p=f(0.5)[:18], u=rng.random(18))
    for far in (np.inf, 1e33, 1e-35):
        check(g, x, f(far), p=f(0.7), u=rng.random(m))
        check(g, x, f(far), f(6000, np.int32), f(0.7), u=rng.random(m))


def test_refusals(g):
    torch = g._torch
    f = lambda *s, dt=torch.float32: torch.ones(*s, dtype=dt, device=g.torch_device)  # noqa: E731
    u, x = f(3, dt=torch.float64), f(3, 10)

    def refused(fn, status=_abi.GQ_ERR_INVALID_ARGUMENT):
        with pytest.raises(GqError) as e:
            fn()
        assert e.value.status == status

    refused(lambda: g.sample_requests(x))  # no random numbers
    refused(lambda: g.sample_requests(x, uniforms=u, rng_state=f(3, dt=torch.int64)))
    refused(lambda: g.sample_requests(x, uniforms=u.float()))
    refused(lambda: g.sample_requests(x, uniforms=u[:2].contiguous()))
    refused(lambda: g.sample_requests(x, uniforms=u, temperature=f(3, dt=torch.float64)))
    refused(lambda: g.sample_requests(x, uniforms=u, top_k=f(3, dt=torch.int64)))
    refused(lambda: g.sample_requests(x, uniforms=u, top_p=f(6)[::2]))
    refused(lambda: g.sample_requests(x, uniforms=u, min_p=f(2)))
    refused(lambda: g.sample_requests(x.half(), uniforms=u))
    refused(lambda: g.sample_requests(x[0], uniforms=u))
    refused(lambda: g.sample_requests(x, uniforms=u, tokens=f(3, dt=torch.int64)))
    refused(lambda: g.sample_requests(x, uniforms=u.cpu()))
    refused(lambda: g.sample_requests(f(1, 524289), uniforms=u), _abi.GQ_ERR_UNSUPPORTED)
    call, p, t = g.lib.gq_sample_requests, x.data_ptr(), torch.zeros(3, dtype=torch.int32, device=g.torch_device)
    rest = (None, None, None, None, u.data_ptr(), None)
    for bad in ((p, -1, 10, 0, *rest, t.data_ptr(), None), (p, 3, 0, 0, *rest, t.data_ptr(), None), (p, 3, 10, 9, *rest, t.data_ptr(), None),
                (None, 3, 10, 0, *rest, t.data_ptr(), None), (p, 3, 10, 0, *rest, None, None)):
        assert call(g.ctx, *bad) == _abi.GQ_ERR_INVALID_ARGUMENT
    assert call(g.ctx, p, 0, 10, 0, *rest, t.data_ptr(), None) == _abi.GQ_OK
    assert call(None, p, 3, 10, 0, *rest, t.data_ptr(), None) == _abi.GQ_ERR_INVALID_ARGUMENT
    assert g.lib.gq_sync(g.ctx) == _abi.GQ_OK
