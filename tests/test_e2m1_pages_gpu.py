"""Pages of 4-bit values (GQ_KV_E2M1) and rows read back from pages of any type (needs a B200):
stored bytes and rows read back must equal the definition's; attention over such pages has a
relative L2 error of every request's row of at most 1e-5 against 64 bits, the framework's bound
for f32 products (test_paged_gpu.py says why)."""
import ctypes

import numpy as np
import pytest

import e2m1_ref as ref
from gq import CudaBackend, GqError, _abi
from numerics import rel_l2

pytestmark = pytest.mark.gpu

ATTN_REL_L2 = 1e-5


@pytest.fixture(scope="module")
def g():
    be = CudaBackend(0)
    yield be
    be.close()


def dev(g, a):
    return g._torch.from_numpy(np.ascontiguousarray(a)).to(g.torch_device)


def hard_rows(rng, n, width):
    """Numbers where a rounding can go wrong, a kind for each block of 16."""
    x = rng.standard_normal((n, width // 16, 16)).astype(np.float32)
    kind = rng.integers(0, 12, x.shape[:2])
    for i, j in np.argwhere(kind > 2):
        b = x[i, j]
        k = kind[i, j]
        if k == 3:  # few bits: many middles
            x[i, j] = np.round(b * 4) / 4
        elif k == 4:  # the middles of codes under a given scale, and the numbers beside them
            s = ref.SCALES[rng.integers(1, 127)]
            mid = rng.choice([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], 16) * s
            mid[0] = 6 * s
            x[i, j] = np.nextafter(mid.astype(np.float32), rng.choice([0, np.inf], 16).astype(np.float32)) if rng.random() < 0.5 else mid
            x[i, j] *= rng.choice([-1, 1], 16)
        elif k == 5:  # the middle of two scales, and the numbers beside it
            t = rng.integers(0, 126)
            top = np.float32(3 * (ref.SCALES[t] + ref.SCALES[t + 1]))
            x[i, j] = b / np.abs(b).max() * top * 0.9
            x[i, j, rng.integers(16)] = rng.choice([top, np.nextafter(top, np.float32(0)), np.nextafter(top, np.float32(9e9))])
        elif k == 6:
            x[i, j] = b * np.float32(10.0 ** rng.uniform(-44, 38))
        elif k == 7:
            x[i, j] = rng.choice([0.0, -0.0], 16)
        elif k == 8:
            x[i, j, rng.integers(16)] = rng.choice([np.inf, -np.inf])
        elif k == 9:
            x[i, j, rng.integers(16)] = np.nan
        elif k == 10:
            x[i, j, rng.integers(16)] = 3.4e38
        elif k == 11:
            x[i, j] = b * np.float32(2.0 ** -rng.integers(7, 14))
    return x.reshape(n, width)


SHAPES = [(1, 256, 16), (1, 512, 64), (4, 128, 32), (3, 16, 1), (2, 48, 7), (8, 64, 16), (5, 176, 3), (1, 16, 5)]  # heads, dim, page


@pytest.mark.parametrize("heads,dim,ps", SHAPES)
@pytest.mark.parametrize("scale", [1.0, 1 / 32, 0.037])
def test_append_stores_the_definitions_bytes(g, heads, dim, ps, scale):
    torch = g._torch
    rng = np.random.default_rng(heads * dim + ps)
    n = 150
    pages = -(-n // ps) + 4
    row = dim // 16 * 9
    pool = [rng.integers(0, 256, (pages, heads, ps, row), dtype=np.uint8) for _ in range(2)]
    x = [hard_rows(rng, n, heads * dim) for _ in range(2)]
    slots = rng.permutation(pages * ps)[:n]
    slots[rng.random(n) < 0.1] = -1
    slots[5] = -(2 ** 40)
    d = [dev(g, p) for p in pool]
    wide = torch.zeros(n, heads * dim + 20, device=g.torch_device)  # rows of k lie apart
    wide[:, :heads * dim] = dev(g, x[0])
    g.paged_append(g.kv_pages(*d, k_scale=scale, v_scale=scale), wide[:, :heads * dim], dev(g, x[1]), dev(g, slots))
    g.flush()
    for p, got, rows in zip(pool, d, x):
        with np.errstate(over="ignore"):
            want = ref.encode(rows.reshape(n, heads, dim), scale)
        at = slots >= 0
        p[slots[at] // ps, :, slots[at] % ps] = want[at]
        bad = np.argwhere(got.cpu().numpy() != p)
        assert not len(bad), (bad[:5], len(bad))


def test_every_scale_and_code_stands_for_its_value(g):
    """All 256 scale bytes with all 16 codes, through the read."""
    torch = g._torch
    codes = np.tile(np.arange(16, dtype=np.uint8), (256, 1))
    rows = np.concatenate([codes[:, 0::2] | (codes[:, 1::2] << 4), np.arange(256, dtype=np.uint8)[:, None]], 1)
    pool = dev(g, rows.reshape(16, 1, 16, 9))
    k, v = g.paged_read(g.kv_pages(pool, pool, 0.5, 2.0), torch.arange(256, device=g.torch_device))
    want = ref.decode(rows)
    assert np.array_equal(k.cpu().numpy()[:, 0], (want * 0.5).astype(np.float32), equal_nan=True)
    assert np.array_equal(v.cpu().numpy()[:, 0], (want * 2.0).astype(np.float32), equal_nan=True)


@pytest.mark.parametrize("heads,dim", [(1, 512), (2, 48), (1, 16), (3, 256)])
@pytest.mark.parametrize("pad,skip", [(0, 0), (8, 0), (4, 0), (0, 4), (16, 8)])
def test_rows_of_every_alignment(g, heads, dim, pad, skip):
    """Rows of f32 that begin on 16 or on 32 bytes and lie any multiple of 4 values apart."""
    torch = g._torch
    rng = np.random.default_rng(dim + pad)
    n, ps, row = 70, 8, heads * dim
    x = [hard_rows(rng, n, row) for _ in range(2)]
    slots = dev(g, rng.permutation(12 * ps)[:n])
    pool = [torch.zeros(12, heads, ps, dim // 16 * 9, dtype=torch.uint8, device=g.torch_device) for _ in range(2)]
    stores = [torch.full((n * (row + pad) + skip,), 7.0, device=g.torch_device) for _ in range(4)]
    rows = [t[skip:].view(n, row + pad)[:, :row] for t in stores]
    for i in range(2):
        rows[i].copy_(dev(g, x[i]))
    pages = g.kv_pages(*pool)
    g.paged_append(pages, rows[0], rows[1], slots)
    g.paged_read(pages, slots, k_out=rows[2], v_out=rows[3])
    g.flush()
    with np.errstate(over="ignore"):
        for i in range(2):
            want = ref.decode(ref.encode(x[i].reshape(n, heads, dim), 1.0)).astype(np.float32).reshape(n, row)
            assert np.array_equal(rows[2 + i].cpu().numpy(), want, equal_nan=True)
            kept = stores[2 + i].clone()
            kept[skip:].view(n, row + pad)[:, :row] = 7.0
            assert bool((kept == 7.0).all())


@pytest.mark.parametrize("typ", ["f32", "f16", "bf16", "e4m3", "e2m1"])
@pytest.mark.parametrize("heads,dim,ps", [(1, 256, 16), (1, 512, 64), (4, 128, 32), (3, 16, 1), (2, 48, 7), (1, 64, 16), (7, 112, 3)])
def test_read_gives_the_rows(g, typ, heads, dim, ps):
    torch = g._torch
    rng = np.random.default_rng(dim + ps)
    dt = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "e4m3": torch.float8_e4m3fn}.get(typ)
    pages, n = 9, 133
    if typ == "e2m1":
        both = rng.integers(0, 256, (pages, 2, heads, ps, dim // 16 * 9), dtype=np.uint8)  # keys and values page by page
        values = ref.decode(both)
        both = dev(g, both)
    else:
        both = torch.from_numpy(rng.standard_normal((pages, 2, heads, ps, dim)).astype(np.float32)).to(g.torch_device).to(dt)
        values = both.cpu().float().numpy().astype(np.float64)
    scales = (0.25, 1 / 3) if typ in ("e4m3", "e2m1") else (1.0, 1.0)
    slots = rng.integers(0, pages * ps, n)  # some of them twice
    slots[rng.random(n) < 0.15] = -3
    k = torch.full((n, heads * dim + 8), 7.0, device=g.torch_device)
    v = torch.full((n, heads, dim), 7.0, device=g.torch_device)
    kv = both[:, 0], both[:, 1]
    if kv[1].data_ptr() % 16:  # (a small row's bytes: pools must begin at a multiple of 16)
        with pytest.raises(GqError):
            g.paged_read(g.kv_pages(*kv, *scales), dev(g, slots), k_out=k[:, :heads * dim], v_out=v)
        kv = kv[0].contiguous(), kv[1].contiguous()
    desc = g.kv_pages(*kv, *scales)
    g.paged_read(desc, dev(g, slots), k_out=k[:, :heads * dim], v_out=v)
    g.flush()
    assert bool((k[:, heads * dim:] == 7.0).all())
    for i, (got, s) in enumerate(((k[:, :heads * dim].reshape(n, heads, dim), scales[0]), (v, scales[1]))):
        # (code * scale is exact; the pool's scale rounds once)
        want = values[:, i].astype(np.float32) * np.float32(s)
        want = np.where((slots >= 0)[:, None, None], want[slots // ps, :, slots % ps], np.float32(7.0))
        assert np.array_equal(got.cpu().numpy(), want, equal_nan=True)


def test_slots_past_the_pool_are_reported(g):
    torch = g._torch
    pool = torch.zeros(4, 1, 16, 144, dtype=torch.uint8, device=g.torch_device)
    pages = g.kv_pages(pool[:3], pool[:3].clone())
    rows = torch.full((3, 1, 256), 1.5, device=g.torch_device)  # 6 times a scale of 1/4
    slots = dev(g, np.array([1, 48, 2], np.int64))
    g.paged_append(pages, rows, rows, slots)
    assert g.lib.gq_sync(g.ctx) == _abi.GQ_ERR_DEVICE
    assert g.lib.gq_sync(g.ctx) == _abi.GQ_OK
    assert int(pool[3].sum()) == 0
    k, v = g.paged_read(pages, slots)
    assert g.lib.gq_sync(g.ctx) == _abi.GQ_ERR_DEVICE
    assert k[:, 0, 0].tolist() == [1.5, 0.0, 1.5] and v[:, 0, 5].tolist() == [1.5, 0.0, 1.5]


# ---- attention ----------------------------------------------------------------------------------------


def pools_of(rng, pages, heads, ps, dim):
    x = rng.standard_normal((2, pages, heads, ps, dim)).astype(np.float32)
    x *= np.exp(rng.standard_normal((2, pages, heads, ps, 1)) * 0.5).astype(np.float32)
    return ref.encode(x, 1 / 32)


def attention_ref(q, k, v, table, lens, scale, window, cap, ps):
    """k, v: the values [page, head, row, dim] in f64."""
    b, hq, d = q.shape
    hkv = k.shape[1]
    out = np.zeros((b, hq, d))
    for i in range(b):
        n = min(max(int(lens[i]), 0), table.shape[1] * ps)
        lo = max(0, n - window) if window else 0
        at = np.arange(lo, n)
        if not len(at):
            continue
        ids = table[i, at // ps]
        for h in range(hkv):
            heads = slice(h * (hq // hkv), (h + 1) * (hq // hkv))
            s = q[i, heads].astype(np.float64) @ k[ids, h, at % ps].T * scale
            if cap:
                s = cap * np.tanh(s / cap)
            p = np.exp(s - s.max(1, keepdims=True))
            out[i, heads] = (p / p.sum(1, keepdims=True)) @ v[ids, h, at % ps]
    return out.reshape(b, hq * d)


ATTN = [  # lens, dim, hq, hkv, page, window, cap
    ([1], 256, 8, 1, 16, 0, 0.0), ([0], 256, 8, 1, 16, 0, 0.0), ([333], 256, 8, 1, 16, 512, 0.0), ([700], 256, 8, 1, 16, 512, 0.0),
    ([1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 0, 300], 256, 8, 1, 16, 0, 0.0),
    ([1, 40, 0, 1000, 129, 64, 2000], 512, 8, 1, 16, 0, 0.0), ([5, 77, 600, 0, 1200], 512, 8, 1, 64, 513, 30.0),
    ([50, 90, 1, 0, 511, 512, 513], 128, 16, 4, 32, 0, 50.0), ([100, 3, 40], 128, 4, 4, 16, 17, 0.0), ([9000], 128, 8, 8, 64, 0, 0.0),
    ([200, 1, 1500, 16], 64, 8, 2, 16, 0, 0.0), ([33, 900], 64, 24, 2, 32, 100, 20.0), ([130, 7], 64, 1, 1, 8, 0, 0.0),
    ([30, 250, 1], 256, 12, 1, 128, 0, 0.0), ([1027, 40], 512, 16, 1, 256, 0, 0.0), ([6, 1100], 256, 64, 1, 32, 1000, 0.0),
    ([20, 0, 129], 48, 6, 3, 16, 0, 0.0), ([77, 1], 16, 8, 1, 1, 0, 0.0), ([200, 65], 256, 8, 1, 24, 0, 0.0),
    ([70, 5], 176, 4, 2, 7, 50, 0.0), ([40, 500], 512, 5, 5, 4, 0, 0.0), ([21000, 3, 9000], 256, 8, 1, 16, 0, 0.0),
    ([15000, 0, 8001], 512, 8, 1, 64, 0, 0.0), ([30000] + [10] * 40, 128, 8, 1, 16, 0, 0.0), ([64] * 300, 256, 8, 1, 16, 0, 0.0),
    ([100] * 150, 128, 8, 8, 16, 40, 0.0), ([3000] * 9, 64, 8, 4, 64, 0, 0.0), (list(range(257)), 512, 8, 1, 32, 0, 0.0)]


@pytest.mark.parametrize("lens,dim,hq,hkv,ps,window,cap", ATTN)
def test_attention_matches_64_bits(g, lens, dim, hq, hkv, ps, window, cap):
    torch = g._torch
    rng = np.random.default_rng(len(lens) * 1000 + dim + ps)
    lens = np.array(lens, np.int32)
    need = -(-lens // ps)
    width = int(need.max()) + 2
    n_pages = int(need.sum()) + 3
    k, v = pools_of(rng, n_pages, hkv, ps, dim)
    perm = rng.permutation(n_pages).astype(np.int32)
    table = np.full((len(lens), width), 2 ** 30, np.int32)  # entries that no length reaches are never looked at
    at = 0
    for b, c in enumerate(need):
        table[b, :c] = perm[at:at + c]
        at += c
        if lens[b] % ps:  # rows past the length hold anything: not numbers here
            for pool in (k, v):
                pool[table[b, c - 1], :, lens[b] % ps:] = 255
    q = (2 * rng.standard_normal((len(lens), hq, dim))).astype(np.float32)
    scale = dim ** -0.5
    out = torch.full((len(lens), hq * dim), 5.0, device=g.torch_device)
    pages = g.kv_pages(dev(g, k), dev(g, v), 1 / 32, 1 / 32)
    args = (pages, dev(g, q), dev(g, table), dev(g, lens))
    kw = dict(scale=scale, sliding_window=window, attn_softcap=cap)
    g.paged_attention(*args, **kw, out=out)
    again = g.paged_attention(*args, **kw)
    g.flush()
    got = out.cpu().numpy()
    want = attention_ref(q, ref.decode(k, 1 / 32), ref.decode(v, 1 / 32), table, lens, scale, window, cap, ps)
    for b in range(len(lens)):
        if lens[b] == 0:
            assert not got[b].any()
        else:
            assert rel_l2(got[b], want[b]) <= ATTN_REL_L2, (b, lens[b], rel_l2(got[b], want[b]))
    assert torch.equal(out, again.data)  # the same from run to run


@pytest.mark.parametrize("dim,hq,hkv,ps", [(256, 8, 1, 16), (512, 8, 1, 64), (128, 8, 2, 32), (64, 8, 1, 16), (48, 4, 2, 16)])
def test_constant_values_and_large_scores(g, dim, hq, hkv, ps):
    """The mean of a constant is that constant; scores of hundreds, where one key has all the weight."""
    torch = g._torch
    rng = np.random.default_rng(dim)
    n = 1111
    pages = -(-n // ps)
    k, _ = pools_of(rng, pages, hkv, ps, dim)
    v = ref.encode(np.full((pages, hkv, ps, dim), 1.5, np.float32), 1.0)
    table, lens = np.arange(pages, dtype=np.int32)[None], np.array([n], np.int32)
    q = (100 * rng.standard_normal((1, hq, dim))).astype(np.float32)
    out = g.paged_attention(g.kv_pages(dev(g, k), dev(g, v), 1 / 32, 1.0), dev(g, q), dev(g, table), dev(g, lens), scale=1.0)
    # (1100 weights and products in f32: their sums' roundings are shared by the mean's two sums, but for 2^-20)
    assert np.abs(out.data.cpu().numpy() - 1.5).max() <= 1.5 * 2 ** -19
    v = pools_of(rng, pages, hkv, ps, dim)[1]
    out = g.paged_attention(g.kv_pages(dev(g, k), dev(g, v), 1 / 32, 1 / 32), dev(g, q), dev(g, table), dev(g, lens), scale=1.0)
    want = attention_ref(q, ref.decode(k, 1 / 32), ref.decode(v, 1 / 32), table, lens, 1.0, 0, 0.0, ps)
    # a score of some thousands is off by 2^-21 of the sum of its products' sizes, which is the error of a weight
    size = np.abs(q).max() * np.abs(ref.decode(k, 1 / 32)).max() * dim * 2 ** -21
    assert rel_l2(out.data.cpu().numpy(), want) <= max(ATTN_REL_L2, size)


def test_bad_pages_and_lengths_are_reported(g):
    torch = g._torch
    rng = np.random.default_rng(5)
    for dim, ps in ((256, 16), (512, 64), (128, 32), (48, 16)):
        k, v = pools_of(rng, 6, 1, ps, dim)
        q = rng.standard_normal((2, 8, dim)).astype(np.float32)
        table = np.array([[0, 1, 2], [3, 99, 4]], np.int32)
        lens = np.array([2 * ps + 3, 3 * ps], np.int32)
        pages = g.kv_pages(dev(g, k), dev(g, v), 1 / 32, 1 / 32)
        out = g.paged_attention(pages, dev(g, q), dev(g, table), dev(g, lens), scale=0.1)
        assert g.lib.gq_sync(g.ctx) == _abi.GQ_ERR_DEVICE
        kd, vd = ref.decode(k, 1 / 32), ref.decode(v, 1 / 32)
        zero = np.zeros_like(kd[:1])  # a page outside the pool counts as rows of zeros
        table[1, 1] = 6
        want = attention_ref(q, np.concatenate([kd, zero]), np.concatenate([vd, zero]), table, lens, 0.1, 0, 0.0, ps)
        assert rel_l2(out.data.cpu().numpy(), want) <= ATTN_REL_L2
        table[1, 1], lens[1] = 5, 4 * ps  # past the table's row: cut to it
        out = g.paged_attention(pages, dev(g, q), dev(g, table), dev(g, lens), scale=0.1)
        assert g.lib.gq_sync(g.ctx) == _abi.GQ_ERR_DEVICE
        lens[1] = 3 * ps
        want = attention_ref(q, kd, vd, table, lens, 0.1, 0, 0.0, ps)
        assert rel_l2(out.data.cpu().numpy(), want) <= ATTN_REL_L2
    assert g.lib.gq_sync(g.ctx) == _abi.GQ_OK


def test_pages_apart_and_unaligned(g):
    """Pages of several layers in one allocation: any distance between pages, in bytes."""
    torch = g._torch
    rng = np.random.default_rng(6)
    dim, ps, hkv = 256, 16, 1
    k, v = pools_of(rng, 5, hkv, ps, dim)
    for apart in (2304 + 16, 2304 + 5, 3 * 2304):
        store = torch.zeros(2, 5 * apart, dtype=torch.uint8, device=g.torch_device)
        views = [s.as_strided((5, hkv, ps, 144), (apart, 2304, 144, 1)) for s in (store[0], store[1])]
        if store[1].data_ptr() % 16:
            continue
        for view, pool in zip(views, (k, v)):
            view.copy_(dev(g, pool))
        q = rng.standard_normal((1, 8, dim)).astype(np.float32)
        table, lens = np.array([[3, 0, 4, 1]], np.int32), np.array([61], np.int32)
        pages = g.kv_pages(*views, 1 / 32, 1 / 32)
        out = g.paged_attention(pages, dev(g, q), dev(g, table), dev(g, lens), scale=0.1)
        want = attention_ref(q, ref.decode(k, 1 / 32), ref.decode(v, 1 / 32), table, lens, 0.1, 0, 0.0, ps)
        assert rel_l2(out.data.cpu().numpy(), want) <= ATTN_REL_L2
        rows, _ = g.paged_read(pages, torch.arange(80, device=g.torch_device))
        assert np.array_equal(rows.cpu().numpy()[:, 0], ref.decode(k, 1 / 32)[:, 0].reshape(80, dim).astype(np.float32))


def test_written_attended_and_read_together_in_a_graph():
    """A step's rows written, attended and read back, recorded and replayed on a stream of its own,
    beside another context that does the same."""
    contexts = [CudaBackend(0, own_stream=True) for _ in range(2)]
    torch = contexts[0]._torch
    rng = np.random.default_rng(8)
    dim, ps, n = 256, 16, 40
    work = []
    for g in contexts:
        k, v = pools_of(rng, 12, 1, ps, dim)
        s = dict(k=dev(g, k), v=dev(g, v), q=dev(g, rng.standard_normal((3, 8, dim)).astype(np.float32)),
                 new=[torch.zeros(3, 1, dim, device=g.torch_device) for _ in range(2)],
                 slots=torch.zeros(3, dtype=torch.int64, device=g.torch_device), lens=torch.zeros(3, dtype=torch.int32, device=g.torch_device),
                 table=dev(g, np.arange(12, dtype=np.int32).reshape(3, 4)), out=torch.zeros(3, 8 * dim, device=g.torch_device),
                 rows=[torch.zeros(3, 1, dim, device=g.torch_device) for _ in range(2)])
        s["pages"] = g.kv_pages(s["k"], s["v"], 1 / 32, 1 / 32)
        torch.cuda.synchronize()

        def step(g=g, s=s):
            g.paged_append(s["pages"], *s["new"], s["slots"])
            g.paged_attention(s["pages"], s["q"], s["table"], s["lens"], scale=0.1, out=s["out"])
            g.paged_read(s["pages"], s["slots"], k_out=s["rows"][0], v_out=s["rows"][1])

        step()
        g.flush()
        s["graph"] = g.record(step)
        work.append((g, s, k, v))
    for i in range(n):
        for g, s, k, v in work:
            lens = np.array([i + 1, (7 * i) % 64 + 1, 64 - i], np.int32)
            slots = np.arange(3) * 64 + lens - 1
            rows = rng.standard_normal((2, 3, 1, dim)).astype(np.float32)
            for d, h in ((s["lens"], lens), (s["slots"], slots), (s["new"][0], rows[0]), (s["new"][1], rows[1])):
                d.copy_(dev(g, h))
            for pool, r in zip((k, v), rows):
                pool[slots // ps, :, slots % ps] = ref.encode(r, 1 / 32)
            s["lens_h"], s["slots_h"] = lens, slots
        torch.cuda.synchronize()
        for g, s, _, _ in work:
            g.replay(s["graph"])
        for g, s, k, v in work:
            g.flush()
            kd, vd = ref.decode(k, 1 / 32), ref.decode(v, 1 / 32)
            want = attention_ref(s["q"].cpu().numpy(), kd, vd, s["table"].cpu().numpy(), s["lens_h"], 0.1, 0, 0.0, ps)
            assert rel_l2(s["out"].cpu().numpy(), want) <= ATTN_REL_L2
            for got, values in zip(s["rows"], (kd, vd)):
                assert np.array_equal(got.cpu().numpy(), values[s["slots_h"] // ps, :, s["slots_h"] % ps].astype(np.float32))
    for g, s, _, _ in work:
        g.destroy_graph(s["graph"])
        g.close()


def test_refusals(g):
    torch = g._torch
    u8 = lambda *s: torch.zeros(*s, dtype=torch.uint8, device=g.torch_device)  # noqa: E731

    def refused(fn, status=_abi.GQ_ERR_INVALID_ARGUMENT):
        with pytest.raises(GqError) as e:
            fn()
        assert e.value.status == status

    refused(lambda: g.kv_pages(u8(4, 1, 16, 128), u8(4, 1, 16, 128)))  # no room for scales
    refused(lambda: g.kv_pages(u8(4, 1, 16, 144), torch.zeros(4, 1, 16, 144, device=g.torch_device)), _abi.GQ_ERR_UNSUPPORTED)
    pages = g.kv_pages(u8(4, 2, 16, 144), u8(4, 2, 16, 144))
    slots, rows = torch.zeros(3, dtype=torch.int64, device=g.torch_device), torch.zeros(3, 2, 256, device=g.torch_device)
    refused(lambda: g.paged_read(pages, slots, k_out=rows[:, :1].contiguous(), v_out=rows))
    refused(lambda: g.paged_read(pages, slots.int()))
    refused(lambda: g.paged_read(pages, slots, k_out=torch.zeros(2, 3, 256, device=g.torch_device), v_out=rows))
    refused(lambda: g.paged_read(pages, slots, k_out=rows.half(), v_out=rows))
    unaligned = torch.zeros(3 * 512 + 1, device=g.torch_device)[1:].view(3, 2, 256)
    refused(lambda: g.paged_read(pages, slots, k_out=unaligned, v_out=rows))
    refused(lambda: g.paged_attention(g.kv_pages(u8(1, 1, 16, 297), u8(1, 1, 16, 297)), torch.zeros(1, 8, 528, device=g.torch_device),
                                      torch.zeros(1, 1, dtype=torch.int32, device=g.torch_device),
                                      torch.ones(1, dtype=torch.int32, device=g.torch_device)), _abi.GQ_ERR_UNSUPPORTED)  # head_dim 528
    read = g.lib.gq_paged_read
    st = _abi.KvPagesStruct(pages.k.data_ptr(), pages.v.data_ptr(), 4, 16, 2, 256, 0, _abi.GQ_KV_E2M1, 1.0, 1.0)
    call = lambda p, *a: read(g.ctx, ctypes.addressof(p) if p else None, slots.data_ptr(), *a)  # noqa: E731
    r = rows.data_ptr()
    assert call(st, 3, r, r, 0, 0) == _abi.GQ_OK
    assert call(None, 3, r, r, 0, 0) == _abi.GQ_ERR_INVALID_ARGUMENT
    for bad in ((-1, r, r, 0, 0), (3, None, r, 0, 0), (3, r, r, 508, 0), (3, r, r, 0, 514)):
        assert call(st, *bad) == _abi.GQ_ERR_INVALID_ARGUMENT
    for field, value, status in (("head_dim", 264, _abi.GQ_ERR_UNSUPPORTED), ("page_stride", 16 * 2 * 144 - 1, _abi.GQ_ERR_INVALID_ARGUMENT),
                                 ("type", 5, _abi.GQ_ERR_UNSUPPORTED), ("k_scale", 0.0, _abi.GQ_ERR_INVALID_ARGUMENT)):
        bad = _abi.KvPagesStruct.from_buffer_copy(st)
        setattr(bad, field, value)
        assert call(bad, 3, r, r, 0, 0) == status, field
    assert g.lib.gq_sync(g.ctx) == _abi.GQ_OK
    g.paged_read(pages, slots[:0])  # nothing to do
    g.flush()
