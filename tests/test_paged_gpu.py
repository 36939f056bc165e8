"""The paged key-value cache (gq_paged_reserve, gq_paged_release, gq_paged_append,
gq_paged_attention) against plain implementations in 64 bits (needs a B200).

Whole numbers and stored codes must be equal. Attention: relative L2 error of every
request's row at most 1e-5, the framework's bound for f32 products: with scores of a
few units, an f32 sum of up to 512 products is off by some 1e-6 of a score's size,
which is the relative error of a weight, and the weighted mean of the values carries
it on. Where the values are a constant, the mean is that constant to f32 rounding.
"""
import ctypes
from ctypes import c_void_p

import numpy as np
import pytest

from gq import CudaBackend, GqError, _abi
from numerics import rel_l2

pytestmark = pytest.mark.gpu

TYPES = ["f32", "f16", "bf16", "e4m3"]
ATTN_REL_L2 = 1e-5


@pytest.fixture(scope="module")
def g():
    be = CudaBackend(0)
    yield be
    be.close()


def tdtype(g, name):
    t = g._torch
    return {"f32": t.float32, "f16": t.float16, "bf16": t.bfloat16, "e4m3": t.float8_e4m3fn}[name]


def i32(g, a):
    return g._torch.tensor(np.asarray(a, dtype=np.int32), device=g.torch_device)


def sync_status(g):
    return g.lib.gq_sync(g.ctx)


# ---- reserve and release ------------------------------------------------------------------------------


def reserve_ref(seq, new, ps, table, free, count, max_tokens, n_pages):
    """The definition, token by token."""
    table, seq, new = table.copy(), np.maximum(seq, 0), np.maximum(new, 0)
    have = -(-(seq + new) // ps)
    had = -(-seq // ps)
    slots, pos = np.full(max_tokens, -1, np.int64), np.zeros(max_tokens, np.int32)
    own = np.full(max_tokens, -1, np.int32)
    if (have - had).sum() > count or (len(seq) and have.max() > table.shape[1]) or new.sum() > max_tokens:
        return table, slots, pos, own, seq.astype(np.int32), count, False
    t = 0
    for b in range(len(seq)):
        for p in range(had[b], have[b]):
            count -= 1
            table[b, p] = free[count]
        for i in range(new[b]):
            at = seq[b] + i
            slots[t], pos[t], own[t] = int(table[b, at // ps]) * ps + at % ps, at, b
            t += 1
    return table, slots, pos, own, (seq + new).astype(np.int32), count, True


def pool_state(rng, seq, ps, width, spare):
    """Tables for the given lengths, drawn from a pool, and its free list."""
    need = -(-np.maximum(seq, 0) // ps)
    n = int(need.sum()) + spare
    perm = rng.permutation(n).astype(np.int32)
    table = np.full((len(seq), width), -1, np.int32)
    at = 0
    for b, k in enumerate(need):
        table[b, :k] = perm[at:at + k]
        at += k
    free = np.full(max(n, 1), -1, np.int32)
    free[:spare] = perm[at:]
    return table, free, spare, n


def run_reserve(g, seq, new, ps, table, free, count, max_tokens, alias=False):
    torch = g._torch
    d = dict(seq=i32(g, seq), new=i32(g, new), table=i32(g, table), free=i32(g, free), count=i32(g, [count]))
    d["slots"] = torch.full((max_tokens,), -9, dtype=torch.int64, device=g.torch_device)
    d["pos"], d["own"] = i32(g, np.full(max_tokens, -9)), i32(g, np.full(max_tokens, -9))
    d["tot"] = d["seq"] if alias else i32(g, np.full(len(seq), -9))
    d["left"] = d["count"] if alias else i32(g, [-9])
    g.paged_reserve(d["seq"], d["new"], ps, d["table"], d["free"], d["count"], slots=d["slots"], positions=d["pos"],
                    owners=d["own"], totals=d["tot"], free_left=d["left"])
    rc = sync_status(g)
    return {k: v.cpu().numpy() for k, v in d.items()}, rc


RESERVE = [  # batch, page, most old tokens, most new tokens, padding
    (1, 16, 0, 1, 0), (1, 1, 5, 3, 2), (3, 7, 50, 30, 1), (64, 16, 400, 1, 0), (65, 16, 4000, 1, 7),
    (513, 32, 100, 40, 5), (1300, 16, 3, 2, 0), (40, 64, 1000, 4000, 11), (16384, 16, 40, 2, 3)]


@pytest.mark.parametrize("batch,ps,most,most_new,pad", RESERVE)
@pytest.mark.parametrize("alias", [False, True])
def test_reserve_matches_the_definition(g, batch, ps, most, most_new, pad, alias):
    rng = np.random.default_rng(batch * 7 + ps)
    seq = rng.integers(0, most + 1, batch)
    new = rng.integers(0, most_new + 1, batch)
    seq[rng.random(batch) < 0.1] = -3  # an unused place counts as length 0
    new[rng.random(batch) < 0.1] = 0
    width = -(-(most + most_new) // ps) + 2
    need = int((-(-(np.maximum(seq, 0) + new) // ps) - -(-np.maximum(seq, 0) // ps)).sum())
    table, free, count, n = pool_state(rng, seq, ps, width, need + 3)
    tokens = int(new.sum()) + pad
    want = reserve_ref(seq, new, ps, table, free, count, tokens, n)
    got, rc = run_reserve(g, seq, new, ps, table, free, count, tokens, alias)
    assert rc == _abi.GQ_OK and want[6]
    for name, w in zip(("table", "slots", "pos", "own", "tot"), want):
        np.testing.assert_array_equal(got[name], w, err_msg=name)
    assert got["left"][0] == want[5]


@pytest.mark.parametrize("why", ["pool", "row", "tokens", "count"])
def test_reserve_is_all_or_nothing(g, why):
    rng = np.random.default_rng(5)
    seq, new, ps = np.array([17, 0, 40]), np.array([20, 5, 1]), 16
    table, free, count, _ = pool_state(rng, seq, ps, 4, 1 if why == "pool" else 9)  # two pages are needed
    if why == "row":
        table = np.ascontiguousarray(table[:, :2])  # the first request needs three entries
    listed = len(free) + 4 if why == "count" else count
    tokens = 25 if why == "tokens" else 26
    got, rc = run_reserve(g, seq, new, ps, table, free, listed, tokens)
    assert rc == _abi.GQ_ERR_DEVICE and b"paged" in g.lib.gq_last_error(g.ctx)
    np.testing.assert_array_equal(got["table"], table)
    assert (got["slots"] == -1).all() and (got["own"] == -1).all() and (got["pos"] == 0).all()
    np.testing.assert_array_equal(got["tot"], seq)
    assert got["left"][0] == min(listed, len(free))
    assert sync_status(g) == _abi.GQ_OK  # reported once


def test_reserve_refuses_ids_outside_the_pool(g):
    table, free = np.array([[7, -1, -1]], np.int32), np.array([1, 99, 0], np.int32)
    got, rc = run_reserve(g, [3], [20], 8, table, free, 3, 20)  # pages 7 (outside: 3 pages), 0 and 99 (outside)
    assert rc == _abi.GQ_ERR_DEVICE
    np.testing.assert_array_equal(got["slots"], [-1] * 5 + list(range(8)) + [-1] * 7)


def test_release_undoes_reserve(g):
    rng = np.random.default_rng(11)
    torch = g._torch
    for batch, ps in ((1, 16), (33, 16), (700, 3), (16384, 8)):
        seq, new = rng.integers(0, 60, batch), rng.integers(0, 50, batch)
        width = 120 // ps + 2
        table, free, count, n = pool_state(rng, seq, ps, width, batch * (50 // ps + 2))
        got, rc = run_reserve(g, seq, new, ps, table, free, count, int(new.sum()))
        assert rc == _abi.GQ_OK
        lens, left, pool = i32(g, got["tot"]), i32(g, got["left"]), i32(g, got["free"])
        pool[int(got["left"][0]):count] = -5  # what was taken from the list is no longer in it
        g.paged_release(lens, i32(g, seq), ps, i32(g, got["table"]), pool, left, totals=lens, free_left=left)
        assert sync_status(g) == _abi.GQ_OK
        np.testing.assert_array_equal(pool.cpu().numpy(), free)
        assert int(left[0]) == count
        np.testing.assert_array_equal(lens.cpu().numpy(), seq)


def test_release_keeps_and_ends(g):
    ps = 4
    table = np.array([[0, 1, 2], [3, 4, -1], [5, -1, -1]], np.int32)
    free = np.array([6, 7, -1, -1, -1, -1, -1, -1], np.int32)
    lens, keep = np.array([10, 8, -2]), np.array([4, 100, 0])
    pool, left, tot = i32(g, free), i32(g, [-9]), i32(g, [-9] * 3)
    g.paged_release(i32(g, lens), i32(g, keep), ps, i32(g, table), pool, i32(g, [2]), totals=tot, free_left=left)
    assert sync_status(g) == _abi.GQ_OK
    np.testing.assert_array_equal(pool.cpu().numpy(), [6, 7, 2, 1, -1, -1, -1, -1])
    np.testing.assert_array_equal(tot.cpu().numpy(), [4, 8, 0])
    assert int(left[0]) == 4
    # a list that would outgrow the pool: nothing is given back
    pool = i32(g, free)
    g.paged_release(i32(g, lens), i32(g, keep), ps, i32(g, table), pool, i32(g, [7]), totals=tot, free_left=left)
    assert sync_status(g) == _abi.GQ_ERR_DEVICE
    np.testing.assert_array_equal(pool.cpu().numpy(), free)
    np.testing.assert_array_equal(tot.cpu().numpy(), [10, 8, 0])
    assert int(left[0]) == 7


# ---- append -------------------------------------------------------------------------------------------


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("t,h,d,ps", [(1, 1, 256, 16), (64, 1, 512, 16), (37, 3, 20, 5), (300, 2, 128, 64), (9, 5, 4, 1)])
def test_append_stores_the_rounded_rows(g, name, t, h, d, ps):
    torch = g._torch
    rng = np.random.default_rng(t + d)
    dt = tdtype(g, name)
    n_pages = -(-2 * t // ps) + 1
    k_scale, v_scale = (0.03125, 0.05) if name == "e4m3" else (1.0, 1.0)
    pools = [torch.zeros(n_pages, h, ps, d, device=g.torch_device).to(dt) for _ in range(2)]
    pages = g.kv_pages(*pools, k_scale=k_scale, v_scale=v_scale)
    x = rng.standard_normal((2, t, h, d)).astype(np.float32) * 8
    x[0, 0, 0, :4] = [np.inf, -np.inf, 1e30, np.nan]  # f16 and e4m3 have no 1e30
    slots = rng.permutation(n_pages * ps)[:t].astype(np.int64)
    slots[t // 2 + 1::5] = -1
    xs = torch.from_numpy(x).to(g.torch_device)
    wide = torch.full((t, h * d + 8), 3.0, device=g.torch_device)  # rows apart
    wide[:, :h * d] = xs[1].reshape(t, -1)
    g.paged_append(pages, xs[0], wide[:, :h * d], torch.from_numpy(slots).to(g.torch_device))
    assert sync_status(g) == _abi.GQ_OK
    for got, rows, scale in ((pools[0], xs[0], k_scale), (pools[1], xs[1], v_scale)):
        want = torch.zeros(n_pages * ps, h, d, device=g.torch_device).to(dt)
        inv = float(np.float32(1.0) / np.float32(scale))
        r = (rows * inv).clamp(-448, 448).to(dt) if name == "e4m3" else rows.to(dt)
        ok = torch.from_numpy(slots >= 0).to(g.torch_device)
        at = torch.from_numpy(slots).to(g.torch_device)[ok]
        want.view(torch.uint8)[at] = r.view(torch.uint8)[ok]
        want = want.view(n_pages, ps, h, d).transpose(1, 2)
        a, b = got.float().cpu().numpy(), want.float().cpu().numpy()
        np.testing.assert_array_equal(np.isnan(a), np.isnan(b))
        np.testing.assert_array_equal(a, b)


def test_append_to_interleaved_pages_and_past_the_pool(g):
    torch = g._torch
    both = torch.zeros(6, 2, 2, 8, 64, device=g.torch_device)  # [page, k or v, head, row, column]
    pages = g.kv_pages(both[:, 0], both[:, 1])
    x = torch.randn(4, 2, 64, device=g.torch_device)
    slots = torch.tensor([47, 0, 48, -1], device=g.torch_device)  # 48 is past the last page
    g.paged_append(pages, x, -x, slots)
    assert sync_status(g) == _abi.GQ_ERR_DEVICE
    want = torch.zeros_like(both)
    want[5, 0, :, 7], want[5, 1, :, 7] = x[0], -x[0]
    want[0, 0, :, 0], want[0, 1, :, 0] = x[1], -x[1]
    assert torch.equal(both, want)


@pytest.mark.parametrize("name", ["f32", "bf16"])
@pytest.mark.parametrize("t,h,d", [(20011, 1, 128), (20011, 3, 20), (5003, 1, 132)])
def test_append_of_more_rows_than_the_grid_takes_at_once(g, name, t, h, d):
    torch = g._torch
    ps, dt = 16, tdtype(g, name)
    n_pages = t // ps + 3
    pools = [torch.zeros(n_pages, h, ps, d, device=g.torch_device).to(dt) for _ in range(2)]
    gen = torch.Generator(device=g.torch_device).manual_seed(t + d)
    xs = torch.randn(2, t, h, d, device=g.torch_device, generator=gen)
    slots = torch.randperm(n_pages * ps, device=g.torch_device, generator=gen)[:t]
    slots[::7] = -1
    g.paged_append(g.kv_pages(*pools), xs[0], xs[1], slots)
    assert sync_status(g) == _abi.GQ_OK
    for got, rows in zip(pools, xs):
        want = torch.zeros(n_pages * ps, h, d, device=g.torch_device).to(dt)
        want[slots[slots >= 0]] = rows[slots >= 0].to(dt)
        assert torch.equal(got, want.view(n_pages, ps, h, d).transpose(1, 2))


# ---- attention ----------------------------------------------------------------------------------------


class Cache:
    """A paged cache with random contents: everything behind the requests' lengths, and
    every page of no request, is NaN."""

    def __init__(self, g, name, lens, hkv, d, ps, seed, interleave=False, spare=3, room=0, dtype_scale=(1 / 32, 1 / 24)):
        torch = g._torch
        rng = np.random.default_rng(seed)
        lens = np.asarray(lens)
        dt = tdtype(g, name)
        width = max(1, -(-max(int(lens.max(initial=0)), room) // ps)) + 1
        table, _, _, n = pool_state(rng, lens, ps, width, spare)
        self.k_scale, self.v_scale = dtype_scale if name == "e4m3" else (1.0, 1.0)
        gen = torch.Generator(device=g.torch_device)
        gen.manual_seed(seed)
        pool = torch.randn(n, 2, hkv, ps, d, generator=gen, device=g.torch_device)
        pool[:, 0] /= self.k_scale
        pool[:, 1] /= self.v_scale
        used = torch.zeros(n, ps, dtype=torch.bool)
        for b, length in enumerate(lens):
            for p in range(-(-max(int(length), 0) // ps)):
                used[table[b, p], :min(ps, int(length) - p * ps)] = True
        used = used.to(g.torch_device)
        self.values = torch.where(used[:, None, None, :, None], pool, torch.full_like(pool, float("nan"))).to(dt)
        if interleave:
            self.k, self.v = self.values[:, 0], self.values[:, 1]
        else:
            self.k, self.v = self.values[:, 0].contiguous(), self.values[:, 1].contiguous()
        self.table_np, self.lens_np, self.ps, self.hkv, self.d = table, lens, ps, hkv, d
        self.table, self.lens = i32(g, table), i32(g, lens)
        self.pages = g.kv_pages(self.k, self.v, k_scale=self.k_scale, v_scale=self.v_scale)

    def rows(self, b, lo, hi):
        """The visible keys and values of request b in 64 bits, [n, hkv, d]."""
        at = np.arange(lo, hi)
        ids = self.table_np[b, at // self.ps]
        k = self.k.float()[ids, :, at % self.ps].double().cpu().numpy() * self.k_scale
        v = self.v.float()[ids, :, at % self.ps].double().cpu().numpy() * self.v_scale
        return k, v


def attend_ref(cache, q, scale, window=0, softcap=0.0):
    q = q.double().cpu().numpy()
    batch, hq, d = q.shape
    group = hq // cache.hkv
    out = np.zeros((batch, hq, d))
    for b, n in enumerate(cache.lens_np):
        if n <= 0:
            continue
        lo = max(0, n - window) if window else 0
        k, v = cache.rows(b, lo, n)
        for h in range(hq):
            s = scale * (k[:, h // group] @ q[b, h])
            if softcap > 0:
                s = softcap * np.tanh(s / softcap)
            p = np.exp(s - s.max())
            out[b, h] = (p @ v[:, h // group]) / p.sum()
    return out.reshape(batch, hq * d)


def check_attend(g, cache, hq, window=0, softcap=0.0, scale=None, seed=3, q=None):
    torch = g._torch
    gen = torch.Generator(device=g.torch_device)
    gen.manual_seed(seed)
    if q is None:
        q = 2.0 * torch.randn(len(cache.lens_np), hq, cache.d, generator=gen, device=g.torch_device)
    scale = cache.d ** -0.5 if scale is None else scale
    out = torch.full((len(cache.lens_np), hq * cache.d), 7.0, device=g.torch_device)
    g.paged_attention(cache.pages, q, cache.table, cache.lens, scale=scale, sliding_window=window, attn_softcap=softcap, out=out)
    assert sync_status(g) == _abi.GQ_OK
    got, want = out.cpu().numpy(), attend_ref(cache, q, scale, window, softcap)
    for b, n in enumerate(cache.lens_np):
        if n <= 0:
            assert (got[b] == 0).all(), f"request {b} has no keys"
        else:
            assert np.isfinite(got[b]).all(), f"request {b} of length {n}"
            err = rel_l2(got[b], want[b])
            assert err <= ATTN_REL_L2, f"request {b} of length {n}: {err:.2e}"
    return out


LENS = [0, 1, 2, 15, 16, 17, 63, 64, 65, 130, 511, 513, 1000, -1]


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("d,hkv,group", [(64, 1, 8), (128, 2, 4), (256, 1, 8), (512, 1, 8), (256, 3, 1), (128, 1, 16), (64, 2, 13)])
@pytest.mark.parametrize("window,softcap", [(0, 0.0), (100, 0.0), (512, 30.0), (3000, 0.0)])
@pytest.mark.parametrize("room", [0, 20000])
def test_attention_lengths_heads_and_types(g, name, d, hkv, group, window, softcap, room):
    """room: tokens the table rows could hold; long rows and windows are cut over the grid,
    short ones go to a cluster each."""
    cache = Cache(g, name, LENS, hkv, d, 16, seed=d + hkv, room=room)
    check_attend(g, cache, hkv * group, window, softcap)


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("d", [4, 8, 20, 80, 96, 192, 320, 508])
def test_attention_other_head_dims(g, name, d):
    check_attend(g, Cache(g, name, [0, 1, 33, 200], 2, d, 16, seed=d), 6, 50 if d == 80 else 0)


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("ps", [1, 3, 4, 8, 16, 24, 32, 64, 100, 128, 256])
@pytest.mark.parametrize("d", [128, 512])
@pytest.mark.parametrize("window", [77, 0])
def test_attention_page_sizes(g, name, ps, d, window):
    check_attend(g, Cache(g, name, [1, 7, 100, 129, 600], 2, d, ps, seed=ps, room=0 if window else 20000), 8, window)


@pytest.mark.parametrize("name", ["f32", "bf16", "e4m3"])
@pytest.mark.parametrize("batch,length", [(1, 1), (1, 40000), (2, 9001), (300, 33)])
def test_attention_splits_and_joins(g, name, batch, length):
    """One long request is cut over every SM and joined in two levels; many short ones
    share CTAs; lengths in between mix cut and whole units."""
    rng = np.random.default_rng(batch)
    lens = rng.integers(1, length + 1, batch)
    lens[0] = length
    cache = Cache(g, name, lens, 1, 256, 16, seed=batch)
    a = check_attend(g, cache, 8)
    assert g._torch.equal(a, check_attend(g, cache, 8))  # a fixed order of sums


def test_attention_of_a_constant_value(g):
    """Weights sum to one: equal values come back, whatever the scores (large ones too)."""
    torch = g._torch
    for name in TYPES:
        cache = Cache(g, name, [1, 17, 300, 5000], 1, 128, 16, seed=1)
        v = torch.where(torch.isnan(cache.v.float()), cache.v.float(), torch.full_like(cache.v.float(), 3.0 / cache.v_scale))
        cache.v.copy_(v.to(cache.v.dtype))
        q = 100.0 * torch.randn(4, 8, 128, device=g.torch_device)
        out = g.paged_attention(cache.pages, q, cache.table, cache.lens, scale=1.0).data
        assert sync_status(g) == _abi.GQ_OK
        # at most one rounding of each product and sum: 5000 terms of 2^-24 each, in any order
        assert float((out - 3.0).abs().max()) <= 3.0 * 5000 * 2.0 ** -24


def test_attention_rising_and_falling_maxima(g):
    """Scores that grow along the cache (each tile raises the maximum) and that shrink."""
    torch = g._torch
    for sign in (1.0, -1.0):
        cache = Cache(g, "f32", [700], 1, 64, 16, seed=4)
        ramp = torch.linspace(-40, 40, 700, device=g.torch_device) * sign
        at = torch.arange(700, device=g.torch_device)
        ids = cache.table[0].long()[at // 16]
        cache.k[ids, 0, at % 16] = 0.0
        cache.k[ids, 0, at % 16, 0] = ramp
        q = torch.zeros(1, 8, 64, device=g.torch_device)
        q[..., 0] = 2.0
        check_attend(g, cache, 8, scale=1.0, q=q)


def test_attention_strided_queries_and_interleaved_pages(g):
    torch = g._torch
    for name in TYPES:
        cache = Cache(g, name, [5, 90, 333], 2, 128, 16, seed=9, interleave=True)
        wide = torch.randn(3, 8 + 4, 128, device=g.torch_device)  # q | k | v of a stacked projection
        check_attend(g, cache, 8, q=wide[:, :8])


def test_attention_in_a_graph_follows_the_device_lengths(g):
    torch = g._torch
    own = CudaBackend(0, own_stream=True)
    cache = Cache(own, "bf16", [700, 40, 0], 1, 256, 16, seed=2)
    q = 2.0 * torch.randn(3, 8, 256, device=own.torch_device)
    out = torch.zeros(3, 8 * 256, device=own.torch_device)
    torch.cuda.synchronize()
    fn = lambda: own.paged_attention(cache.pages, q, cache.table, cache.lens, scale=0.0625, out=out)  # noqa: E731
    fn()
    graph = own.record(fn)
    for lens in ([700, 40, 0], [1, 40, 0], [650, 0, 0]):
        cache.lens.copy_(i32(own, lens))
        torch.cuda.synchronize()
        own.replay(graph)
        own.flush()
        cache.lens_np = np.asarray(lens)
        want = attend_ref(cache, q, 0.0625)
        for b, n in enumerate(lens):
            got = out[b].cpu().numpy()
            assert (got == 0).all() if n == 0 else rel_l2(got, want[b]) <= ATTN_REL_L2
    own.destroy_graph(graph)
    own.close()


def test_a_recorded_call_outlives_larger_ones(g):
    """The memory of the partial results does not move when a later call needs more."""
    torch = g._torch
    own = CudaBackend(0, own_stream=True)
    small = Cache(own, "bf16", [900], 1, 64, 16, seed=21)
    q = torch.randn(1, 4, 64, device=own.torch_device)
    out = torch.zeros(1, 4 * 64, device=own.torch_device)
    fn = lambda: own.paged_attention(small.pages, q, small.table, small.lens, scale=0.125, out=out)  # noqa: E731
    torch.cuda.synchronize()
    fn()
    graph = own.record(fn)
    large = Cache(own, "bf16", [5000] * 40, 1, 512, 16, seed=22)
    torch.cuda.synchronize()
    check_attend(own, large, 8)
    out.zero_()
    torch.cuda.synchronize()
    own.replay(graph)
    own.flush()
    assert rel_l2(out.cpu().numpy(), attend_ref(small, q, 0.125)) <= ATTN_REL_L2
    own.destroy_graph(graph)
    own.close()


def test_attention_reports_bad_pages_and_long_lengths(g):
    torch = g._torch
    cache = Cache(g, "bf16", [40, 40], 1, 128, 16, seed=6)
    q = torch.randn(2, 8, 128, device=g.torch_device)
    ok = g.paged_attention(cache.pages, q, cache.table, cache.lens, scale=0.1).data.clone()
    assert sync_status(g) == _abi.GQ_OK
    for bad in (-1, 10 ** 6):
        table = cache.table.clone()
        table[0, 1] = bad
        got = g.paged_attention(cache.pages, q, table, cache.lens, scale=0.1).data
        assert sync_status(g) == _abi.GQ_ERR_DEVICE
        assert torch.isfinite(got).all() and torch.equal(got[1], ok[1])
        # the page counts as sixteen rows of zeros
        k, v = cache.rows(0, 0, 40)
        k[16:32], v[16:32] = 0, 0
        for h in range(8):
            s = 0.1 * (k[:, 0] @ q[0, h].double().cpu().numpy())
            p = np.exp(s - s.max())
            assert rel_l2(got[0].view(8, 128)[h].cpu().numpy(), p @ v[:, 0] / p.sum()) <= ATTN_REL_L2
    lens = i32(g, [10 ** 6, 40])  # past the table row: cut to it; the row's last page is another request's or none
    table = cache.table.clone()
    table[0, :] = table[1, 0]
    got = g.paged_attention(cache.pages, q, table, lens, scale=0.1).data
    assert sync_status(g) == _abi.GQ_ERR_DEVICE
    assert torch.equal(got[1], ok[1])


def test_refusals(g):
    torch = g._torch
    z = lambda *s, dt=torch.float32: torch.zeros(*s, dtype=dt, device=g.torch_device)  # noqa: E731
    pages = g.kv_pages(z(4, 2, 16, 64), z(4, 2, 16, 64))
    table, lens = i32(g, np.zeros((2, 2))), i32(g, [3, 4])
    q = z(2, 4, 64)

    def refused(fn, status=_abi.GQ_ERR_INVALID_ARGUMENT):
        with pytest.raises(GqError) as e:
            fn()
        assert e.value.status == status
        assert sync_status(g) == _abi.GQ_OK

    refused(lambda: g.kv_pages(z(4, 2, 16, 64), z(4, 2, 16, 32)))
    refused(lambda: g.kv_pages(z(4, 2, 16, 64, dt=torch.int8), z(4, 2, 16, 64, dt=torch.int8)), _abi.GQ_ERR_UNSUPPORTED)
    refused(lambda: g.kv_pages(z(4, 2, 64, 16).transpose(2, 3), z(4, 2, 64, 16).transpose(2, 3)))
    refused(lambda: g.paged_attention(pages, z(2, 3, 64), table, lens))  # 3 query heads over 2
    refused(lambda: g.paged_attention(pages, z(2, 130, 64), table, lens), _abi.GQ_ERR_UNSUPPORTED)
    refused(lambda: g.paged_attention(pages, z(1, 4, 64), table, lens))
    refused(lambda: g.paged_attention(pages, z(2, 4, 32), table, lens))
    refused(lambda: g.paged_attention(pages, q.double(), table, lens))
    refused(lambda: g.paged_attention(pages, q[:1].expand(2, 4, 64), table, lens))  # rows on one another
    refused(lambda: g.paged_attention(pages, q, table.long(), lens))
    refused(lambda: g.paged_attention(pages, q, table[:1], lens))
    refused(lambda: g.paged_attention(pages, q, table, lens, out=z(2, 255)))
    refused(lambda: g.paged_attention(g.kv_pages(z(4, 2, 16, 516), z(4, 2, 16, 516)), z(2, 4, 516), table, lens),
            _abi.GQ_ERR_UNSUPPORTED)
    refused(lambda: g.paged_attention(g.kv_pages(z(4, 2, 16, 64), z(4, 2, 16, 64), k_scale=2.0), q, table, lens))
    refused(lambda: g.paged_append(pages, z(3, 2, 64), z(2, 2, 64), z(3, dt=torch.int64)))
    refused(lambda: g.paged_append(pages, z(3, 2, 64), z(3, 2, 64), z(3, dt=torch.int32)))
    refused(lambda: g.paged_append(pages, z(3, 2, 66)[..., 1:65], z(3, 2, 64), z(3, dt=torch.int64)))
    free, one = i32(g, [0]), i32(g, [1])
    many = i32(g, np.zeros(16385))
    with pytest.raises(GqError) as e:
        g.paged_release(many, many, 16, i32(g, np.zeros((16385, 1))), free, one, totals=many, free_left=one)
    assert e.value.status == _abi.GQ_ERR_UNSUPPORTED
    refused(lambda: g.paged_release(lens, lens, 0, table, free, one, totals=lens, free_left=one))
    refused(lambda: g.paged_release(lens, lens[:1], 16, table, free, one, totals=lens, free_left=one))
    lib = g.lib
    assert lib.gq_paged_attention(g.ctx, None, None, 1, 1, 0, None, 0, None, 1.0, 0, 0.0, None) == _abi.GQ_ERR_INVALID_ARGUMENT
    assert lib.gq_paged_append(None, None, None, None, 0, 0, 0, None) == _abi.GQ_ERR_INVALID_ARGUMENT
    st = _abi.KvPagesStruct(pages.struct.k + 4, pages.struct.v, 4, 16, 2, 64, 0, 0, 1.0, 1.0)  # off 16 bytes
    assert lib.gq_paged_append(g.ctx, ctypes.byref(st), c_void_p(q.data_ptr()), c_void_p(q.data_ptr()), 1, 0, 0,
                               c_void_p(lens.data_ptr())) == _abi.GQ_ERR_INVALID_ARGUMENT


def test_empty_calls(g):
    torch = g._torch
    z = lambda *s, dt=torch.float32: torch.zeros(*s, dtype=dt, device=g.torch_device)  # noqa: E731
    pages = g.kv_pages(z(4, 2, 16, 64), z(4, 2, 16, 64))
    none = i32(g, [])
    assert g.paged_attention(pages, z(0, 4, 64), i32(g, np.zeros((0, 2))), none).data.shape == (0, 256)
    g.paged_append(pages, z(0, 2, 64), z(0, 2, 64), z(0, dt=torch.int64))
    left, count = i32(g, [-9]), i32(g, [1])
    slots, pos = z(2, dt=torch.int64), i32(g, [5, 5])
    g.paged_reserve(none, none, 16, i32(g, np.zeros((0, 2))), i32(g, [0]), count, slots=slots, positions=pos,
                    owners=i32(g, [5, 5]), totals=none, free_left=left)
    assert sync_status(g) == _abi.GQ_OK
    assert int(left[0]) == 1 and slots.tolist() == [-1, -1] and pos.tolist() == [0, 0]
    # no page at all: every length is cut to nothing
    nothing = g.kv_pages(z(0, 2, 16, 64), z(0, 2, 16, 64))
    out = g.paged_attention(nothing, z(1, 4, 64) + 1, i32(g, np.zeros((1, 0))), i32(g, [0])).data
    assert sync_status(g) == _abi.GQ_OK and (out == 0).all()
