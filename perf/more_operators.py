"""More operators of a decode step that serves many requests, and the work they are measured on.

Four operators: key and value rows rounded to 4 bits as they are written into the pages of a cache (`paged_append`), rows of
a cache read back (`paged_read`), attention of one new token of each request over pages of 4-bit values (`paged_attention`),
and tokens drawn from the step's logits with a temperature, top-k, top-p, min-p and random number of each request
(`sample_requests`). `run` computes them in their plain form, in elementary torch operations, or with `own` by the backend's
own calls.

A row of 4-bit values is head_dim / 2 bytes of e2m1 codes (value 2i in the low half of byte i) and then head_dim / 16 bytes
of e4m3 scales, one for every 16 neighbouring values: a value is code * scale of its block * scale of the pool.
"""
import math

import torch

own = False

_GOLDEN = 0.6180339887498949
_DTYPE = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "e4m3": torch.float8_e4m3fn, "e2m1": torch.uint8}
_BITS = {"f32": 32, "f16": 16, "bf16": 16, "e4m3": 8, "e2m1": 4.5}
_CODES = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
_DEV = "cuda"


# ---- the cases ---------------------------------------------------------------------------------------------------


def listed():
    return [
        # one short conversation on a sliding-window layer: the smallest call, where latency is all that counts
        dict(name="attend one", kind="attend", batch=1, max_len=333, hq=8, hkv=1, dim=256, page=16, window=512, softcap=0.0),
        # 64 conversations of every length up to 4096 on a full-attention layer with one key-value head: the ordinary step
        dict(name="attend batch", kind="attend", batch=64, max_len=4096, hq=8, hkv=1, dim=512, page=16, window=0, softcap=0.0),
        # several key-value heads of a smaller size, capped scores, an odd number of requests
        dict(name="attend heads", kind="attend", batch=23, max_len=10007, hq=16, hkv=4, dim=128, page=32, window=0, softcap=50.0),
        # four long documents: few rows, so the length itself has to be split
        dict(name="attend long", kind="attend", batch=4, max_len=131072, hq=8, hkv=1, dim=512, page=64, window=0, softcap=0.0),
        # the new token's key and value of 64 requests, and the rows that later steps will see for them
        dict(name="append step", kind="append", tokens=64, hkv=1, dim=256, page=16),
        # a part of a long prompt: written, and read back for the attention of the prompt's next part
        dict(name="append prompt", kind="append", tokens=16411, hkv=1, dim=512, page=64),
        # the last tokens of a draft, looked at again
        dict(name="read draft", kind="read", tokens=40, hkv=1, dim=256, page=16, type="e2m1"),
        # a long request leaves for another pool
        dict(name="read request", kind="read", tokens=32771, hkv=1, dim=512, page=16, type="e2m1"),
        # one request's token over a large vocabulary
        dict(name="sample one", kind="sample", rows=1, vocab=262144, masked=0),
        # an odd number of requests over a vocabulary of another model's size
        dict(name="sample some", kind="sample", rows=37, vocab=32003, masked=3),
        # 64 requests with settings of their own, some of them under a grammar's mask
        dict(name="sample batch", kind="sample", rows=64, vocab=262144, masked=8),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["attend"] * 5 + ["append"] * 2 + ["read"] * 2 + ["sample"] * 3)
    page = rng.choice([16, 32, 64])
    if kind == "attend":
        dim, hkv, group = rng.choice([64, 128, 256, 256, 512, 512]), rng.choice([1, 1, 2, 4, 8]), rng.choice([1, 2, 4, 8, 8])
        rows = max(64, _log(rng, 2.0e5, 1.4e8) // (2 * hkv * dim * 9 // 16))  # tokens of all requests together
        batch = min(_log(rng, 1, 256), rows)
        return dict(kind=kind, batch=batch, max_len=min(131072, max(1, 2 * rows // batch - 1)), hq=hkv * group, hkv=hkv, dim=dim,
                    page=page, window=rng.choice([0, 0, 512, 1000]), softcap=rng.choice([0.0, 0.0, 50.0]))
    if kind in ("append", "read"):
        dim, hkv = rng.choice([64, 128, 256, 512]), rng.choice([1, 2, 4])
        case = dict(kind=kind, tokens=_log(rng, 1, 16384 * 512 // (dim * hkv)), hkv=hkv, dim=dim, page=page)
        return case if kind == "append" else dict(case, type=rng.choice(["e2m1", "e2m1", "e2m1", "e4m3", "bf16", "f16", "f32"]))
    rows = _log(rng, 1, 128)
    return dict(kind=kind, rows=rows, vocab=_log(rng, 20000, 262144 if rows <= 64 else 131072), masked=rng.choice([0, 2, rows // 3]))


def _spread(n, most, least=1):
    """n whole numbers over [least, most], the same ones for every seed, the most among them."""
    return [most if i == 0 else least + int((most + 1 - least) * ((i * _GOLDEN) % 1.0)) for i in range(n)]


def _ceil(a, b):
    return -(-a // b)


def work(case):
    kind = case["kind"]
    if kind == "attend":
        lens = _spread(case["batch"], case["max_len"])
        keys = [min(n, case["window"]) if case["window"] else n for n in lens]
        pages = sum(_ceil(n, case["page"]) for n in keys)
        return {"bytes": sum(keys) * 2 * case["hkv"] * case["dim"] * 9 // 16 + 8 * case["batch"] * case["hq"] * case["dim"] + 4 * pages
                + 4 * case["batch"], "flops": 4 * sum(keys) * case["hq"] * case["dim"]}
    if kind == "append":  # the rows in, their pages written, and what was written read back
        return {"bytes": case["tokens"] * (2 * case["hkv"] * case["dim"] * (4 + 9 / 16 + 4) + 8), "flops": 0}
    if kind == "read":
        return {"bytes": case["tokens"] * (2 * case["hkv"] * case["dim"] * (_BITS[case["type"]] / 8 + 4) + 8), "flops": 0}
    return {"bytes": case["rows"] * (4 * case["vocab"] + 32), "flops": 4 * case["rows"] * case["vocab"]}


# ---- what a program has in hand --------------------------------------------------------------------------------


def _ints(values, order=None):
    t = torch.tensor(values, dtype=torch.int32)
    return (t if order is None else t[order]).to(_DEV)


def _pages_of(lens, page, width, n_pages, gen):
    """A block table: every request's pages drawn at random from the pool."""
    perm = torch.randperm(n_pages, generator=gen, device=_DEV).to(torch.int32)
    need = (lens.long() + page - 1) // page
    start = need.cumsum(0) - need
    col = torch.arange(width, device=_DEV)
    at = start[:, None] + col[None]
    return torch.where(col[None] < need[:, None], perm[at.clamp(max=n_pages - 1)], torch.full_like(at, -1, dtype=torch.int32)).contiguous()


def _some_rows(shape, gen):
    """Rows of 4-bit values as a cache holds them: random numbers over their block's largest."""
    dim = shape[-1]
    x = torch.randn(*shape[:-1], dim // 16, 16, generator=gen, device=_DEV)
    scale = (x.abs().amax(-1, keepdim=True) * (32 / 6)).to(torch.float8_e4m3fn)
    code = torch.bucketize(x.abs() * 32 / scale.float(), torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], device=_DEV), out_int32=True)
    code = (code + 8 * (x < 0)).to(torch.uint8).reshape(*shape[:-1], dim // 2, 2)
    return torch.cat([code[..., 0] | (code[..., 1] << 4), scale.squeeze(-1).view(torch.uint8)], -1)


def _pool(n_pages, hkv, page, dim, typ, gen):
    """Pages full of keys or values as they come out of their norms."""
    pool = torch.empty(n_pages, hkv, page, dim * 9 // 16 if typ == "e2m1" else dim, dtype=_DTYPE[typ], device=_DEV)
    step = max(1, (32 << 20) // (hkv * page * dim))
    for i in range(0, n_pages, step):
        shape = (min(step, n_pages - i), hkv, page, dim)
        if typ == "e2m1":
            pool[i:i + step] = _some_rows(shape, gen)
        else:
            x = torch.randn(*shape, generator=gen, device=_DEV)
            pool[i:i + step] = ((x * 32).clamp(-448, 448) if typ == "e4m3" else x).to(pool.dtype)
    return pool


def prepare(case, seed):
    gen = torch.Generator(device=_DEV)
    gen.manual_seed(int(seed))
    host = torch.Generator()
    host.manual_seed(int(seed))
    kind, s = case["kind"], {"kind": case["kind"], "case": case}
    # (the scale of the pool: a power of two that leaves room for outliers)
    s["k_scale"], s["v_scale"] = (1 / 32, 1 / 32) if case.get("type", "e2m1") in ("e2m1", "e4m3") else (1.0, 1.0)
    if kind == "attend":
        batch, page, dim, hkv = case["batch"], case["page"], case["dim"], case["hkv"]
        lens = _ints(_spread(batch, case["max_len"]), torch.randperm(batch, generator=host))
        n_pages = int(sum(_ceil(n, page) for n in _spread(batch, case["max_len"]))) + 5
        table = _pages_of(lens, page, _ceil(case["max_len"], page), n_pages, gen)
        last, over = (lens.long() - 1) // page, (lens.long() - 1) % page + 1
        ids = table[torch.arange(batch, device=_DEV), last].long()
        stale = (torch.arange(page, device=_DEV)[None] >= over[:, None])[:, None, :, None]
        for name in ("k", "v"):
            s[name] = _pool(n_pages, hkv, page, dim, "e2m1", gen)
            # what lies behind a request's last token is whatever the memory held: not a number here
            s[name][ids] = torch.where(stale, torch.full_like(s[name][ids], 255), s[name][ids])
        s["q"] = 2.0 * torch.randn(batch, case["hq"], dim, generator=gen, device=_DEV)
        s["out"] = torch.empty(batch, case["hq"] * dim, device=_DEV)
        s.update(lens=lens, table=table, scale=dim ** -0.5, window=case["window"], softcap=case["softcap"])
    elif kind in ("append", "read"):
        n, page, dim, hkv = case["tokens"], case["page"], case["dim"], case["hkv"]
        n_pages = _ceil(n + n // 8, page) + 3
        # requests' tokens lie next to one another in their pages, the pages anywhere
        order = torch.randperm(n_pages, generator=gen, device=_DEV)
        at = torch.arange(n, device=_DEV)
        slots = order[at // page] * page + at % page
        slots[at % 97 == 96] = -1  # places of a padded batch: no row
        s["slots"] = slots
        if kind == "append":
            for name in ("k", "v"):
                s["new_" + name] = torch.randn(n, hkv, dim, generator=gen, device=_DEV)
                s[name] = torch.zeros(n_pages, hkv, page, dim * 9 // 16, dtype=torch.uint8, device=_DEV)
        else:
            for name in ("k", "v"):
                s[name] = _pool(n_pages, hkv, page, dim, case["type"], gen)
        for name in ("k_rows", "v_rows"):  # (places without a row keep what they hold)
            s[name] = torch.zeros(n, hkv, dim, device=_DEV)
    else:
        m, v = case["rows"], case["vocab"]
        logits = 2.5 * torch.randn(m, v, generator=gen, device=_DEV)
        # a few tokens that the context asks for, more of them in some rows than in others
        likely = torch.randint(0, v, (m, 64), generator=gen, device=_DEV)
        logits.scatter_add_(1, likely, 4.0 + 12.0 * torch.rand(m, 64, generator=gen, device=_DEV) ** 2)
        row = torch.arange(m, device=_DEV)
        under = row >= m - case["masked"]  # the last rows follow a grammar that allows one token in 50
        logits.masked_fill_(under[:, None] & (torch.rand(m, v, generator=gen, device=_DEV) > 0.02), -math.inf)
        s["logits"] = logits
        r = torch.rand(m, 4, generator=gen, device=_DEV)
        s["temperature"] = torch.where(row % 8 == 7, torch.zeros(m, device=_DEV), 0.6 + 0.7 * r[:, 0])
        sizes = _ints([64, 0, 40, 0, 1000, 0, 1, 20])
        s["top_k"] = sizes[(row + seed) % 8].contiguous()
        s["top_p"] = torch.where(r[:, 1] < 0.3, torch.ones(m, device=_DEV), 0.8 + 0.19 * r[:, 2])
        s["min_p"] = torch.where(r[:, 3] < 0.6, torch.zeros(m, device=_DEV), 0.1 * r[:, 2])
        s["uniforms"] = torch.rand(m, dtype=torch.float64, generator=gen, device=_DEV)
        s["tokens"] = torch.empty(m, dtype=torch.int32, device=_DEV)
        s["probs"] = torch.empty(m, device=_DEV)
    return s


# ---- the plain forms ---------------------------------------------------------------------------------------------


def _values(rows, dim, scale):
    """The values that rows of codes and scales stand for, in f32."""
    codes = torch.tensor(_CODES + [-c for c in _CODES], device=rows.device)
    packed, scales = rows[..., :dim // 2], rows[..., dim // 2:].contiguous().view(torch.float8_e4m3fn).float()
    v = codes[torch.stack([packed & 15, packed >> 4], -1).reshape(*rows.shape[:-1], dim // 16, 16).int()]
    return (v * scales[..., None] * scale).reshape(*rows.shape[:-1], dim)


def _attend_plain(s):
    k, v, q, lens = s["k"], s["v"], s["q"], s["lens"].long()
    batch, hq, dim = q.shape
    _, hkv, page, _ = k.shape
    ids = s["table"].clamp(min=0).long()
    at = torch.arange(ids.shape[1] * page, device=q.device)
    seen = at[None] < lens[:, None]
    if s["window"]:
        seen = seen & (lens[:, None] - 1 - at[None] < s["window"])
    row = seen[:, None, :, None]
    keys = _values(k[ids], dim, s["k_scale"]).transpose(1, 2).reshape(batch, hkv, -1, dim)
    keys = torch.where(row, keys, torch.zeros_like(keys))
    score = torch.matmul(q.view(batch, hkv, hq // hkv, dim), keys.transpose(2, 3)) * s["scale"]
    if s["softcap"]:
        score = s["softcap"] * torch.tanh(score / s["softcap"])
    del keys
    score = torch.where(seen[:, None, None], score, torch.full_like(score, -math.inf))
    top = score.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    p = torch.exp(score - top)
    total = p.sum(-1, keepdim=True)
    values = _values(v[ids], dim, s["v_scale"]).transpose(1, 2).reshape(batch, hkv, -1, dim)
    values = torch.where(row, values, torch.zeros_like(values))
    out = torch.matmul(p, values) / torch.where(total == 0, torch.ones_like(total), total)
    return out.reshape(batch, hq * dim)


def _nearest(x, least, bits):
    """x rounded to `bits` bits after its first, to whole multiples of 2^(least - bits) below 2^least; ties to even."""
    exponent = (torch.frexp(x)[1] - 1).clamp(least, 8)
    step = torch.tensor([2.0 ** (e - bits) for e in range(least, 9)], dtype=x.dtype, device=x.device)[exponent - least]
    return torch.round(x / step) * step


def _packed(x, scale):
    """Rows of f32 values to rows of codes and scales. In f64: a quotient next to the middle of two codes is not lost."""
    dim = x.shape[-1]
    x = (x * (1.0 / scale)).double().reshape(*x.shape[:-1], dim // 16, 16)
    block = _nearest((x.abs().amax(-1, keepdim=True) / 6).clamp(max=448), -6, 3)
    y = torch.where(block > 0, x.abs() / torch.where(block > 0, block, 1.0), 0.0).clamp(max=6)
    y = _nearest(y, 0, 1)
    code = (y.unsqueeze(-1) > torch.tensor(_CODES[:-1], dtype=torch.float64, device=x.device)).sum(-1) + 8 * torch.signbit(x)
    code = code.to(torch.uint8).reshape(*code.shape[:-2], dim // 2, 2)
    return torch.cat([code[..., 0] | (code[..., 1] << 4), block.squeeze(-1).float().to(torch.float8_e4m3fn).view(torch.uint8)], -1)


def _read_plain(s):
    page, slots = s["k"].shape[2], s["slots"]
    at = slots.clamp(min=0)
    got = {}
    for name in ("k", "v"):
        pool, out = s[name], s[name + "_rows"]
        rows = pool.view(torch.uint8)[at // page, :, at % page].view(pool.dtype) if pool.element_size() == 1 else pool[at // page, :, at % page]
        rows = _values(rows, out.shape[-1], s[name + "_scale"]) if pool.dtype == torch.uint8 else rows.float() * s[name + "_scale"]
        got[name] = torch.where((slots >= 0)[:, None, None], rows, out)
    return got


def _append_plain(s):
    page = s["k"].shape[2]
    take = (s["slots"] >= 0).nonzero().squeeze(1)
    slots = s["slots"][take]
    for name in ("k", "v"):
        s[name][slots // page, :, slots % page] = _packed(s["new_" + name][take], s[name + "_scale"])
    return _read_plain(s)


def _sample_plain(s):
    """In f64: the sums are long, and a random number may fall next to the border of two tokens."""
    l = s["logits"]
    l = torch.where(torch.isnan(l), torch.full_like(l, -math.inf), l)
    m, v = l.shape
    value, order = torch.sort(l, dim=1, descending=True, stable=True)
    top = value[:, :1]
    t = s["temperature"].double()[:, None]
    greedy = t <= 0
    x = torch.where(value == top, 0.0, (value.double() - top.double()) / torch.where(greedy, 1.0, t))
    w = torch.where(value == -math.inf, 0.0, torch.exp(x))
    rank = torch.arange(v, device=l.device)[None]
    k = s["top_k"].long()[:, None]
    kept = (rank < torch.where(k > 0, k, v)) & (~greedy | (rank == 0))
    before = torch.cumsum(torch.where(kept, w, 0.0), 1)
    p = s["top_p"].double()[:, None]
    kept = kept & ((p >= 1) | (before - torch.where(kept, w, 0.0) < p * before[:, -1:]) | (rank == 0))
    kept = kept & (w >= s["min_p"].double()[:, None].clamp(max=1))
    mass = torch.zeros_like(w).scatter_(1, order, torch.where(kept, w, 0.0))
    run = torch.cumsum(mass, 1)
    at = (run <= s["uniforms"][:, None] * run[:, -1:]).sum(1)
    last = torch.where(mass > 0, rank, -1).amax(1)
    token = torch.minimum(at, last)
    prob = torch.where(token >= 0, mass.gather(1, token.clamp(min=0)[:, None])[:, 0] / torch.where(token >= 0, run[:, -1], 1.0), 0.0)
    return {"tokens": token.to(torch.int32), "probs": prob.float()}


# ---- the framework's operators -----------------------------------------------------------------------------------

_backend = []


def _gq():
    if not _backend:
        import os
        import sys
        sys.path.insert(0, os.path.join(os.getcwd(), "gemma-4-webgpu-kernels_b200"))
        from gq import CudaBackend
        _backend.append(CudaBackend(0))
    return _backend[0]


def _pages(s):
    """The description of a layer's pages: made once for a cache, as a program does."""
    if "pages" not in s:
        s["pages"] = _gq().kv_pages(s["k"], s["v"], k_scale=s["k_scale"], v_scale=s["v_scale"])
    return s["pages"]


def _run_own(s):
    g, kind = _gq(), s["kind"]
    if kind == "attend":
        g.paged_attention(_pages(s), s["q"], s["table"], s["lens"], scale=s["scale"], sliding_window=s["window"],
                          attn_softcap=s["softcap"], out=s["out"])
        return s["out"]
    if kind in ("append", "read"):
        if kind == "append":
            g.paged_append(_pages(s), s["new_k"], s["new_v"], s["slots"])
        g.paged_read(_pages(s), s["slots"], k_out=s["k_rows"], v_out=s["v_rows"])
        return {"k": s["k_rows"], "v": s["v_rows"]}
    g.sample_requests(s["logits"], s["temperature"], top_k=s["top_k"], top_p=s["top_p"], min_p=s["min_p"], uniforms=s["uniforms"],
                      tokens=s["tokens"], probs=s["probs"])
    return {"tokens": s["tokens"], "probs": s["probs"]}


_PLAIN = {"attend": _attend_plain, "append": _append_plain, "read": _read_plain, "sample": _sample_plain}


def run(state):
    return _run_own(state) if own else _PLAIN[state["kind"]](state)


# ---- the definitions, in 64 bits ---------------------------------------------------------------------------------


def _exact_values(rows, dim, scale):
    """Sign, exponent and fraction of every code and scale by themselves."""
    packed = rows[..., :dim // 2].long()
    code = torch.stack([packed % 16, packed // 16], -1).flatten(-2)
    size = code % 8
    value = torch.where(size < 2, size * 0.5, (2 + size % 2) * 2.0 ** (size // 2 - 2).double())
    byte = rows[..., dim // 2:].long()
    e, f = (byte // 8) % 16, byte % 8
    s = torch.where(e == 0, f * 2.0 ** -9, (8 + f) * 2.0 ** (e - 10).double())
    return torch.where(code >= 8, -value, value) * s.repeat_interleave(16, -1) * scale


def _exact_rounded(x, scale):
    """What a row of values becomes: every value to the nearest of its block's 15, by its distance to each."""
    codes = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64, device=x.device)
    eights = torch.tensor([(8 + f) * 2.0 ** (e - 10) if e else f * 2.0 ** -9 for e in range(16) for f in range(8)][:127],
                          dtype=torch.float64, device=x.device)
    even = torch.arange(127, device=x.device) % 2

    def nearest(y, grid, odd):
        hi = torch.searchsorted(grid, y).clamp(max=grid.numel() - 1)
        lo = (hi - 1).clamp(min=0)
        up, down = grid[hi] - y, y - grid[lo]
        return torch.where((up < down) | ((up == down) & (odd[hi] == 0)), grid[hi], grid[lo])

    y = (x.double() / scale).unflatten(-1, (-1, 16))
    s = nearest(y.abs().amax(-1, keepdim=True) / 6, eights, even)
    q = nearest(y.abs() / torch.where(s > 0, s, 1.0), codes, even)
    return (torch.sign(y) * q * s * scale).flatten(-2)


def exact(case, seed):
    kind = case["kind"]
    s = prepare(case, seed)
    if kind == "attend":
        page, dim, g = case["page"], case["dim"], case["hq"] // case["hkv"]
        out = torch.zeros(case["batch"], case["hq"], dim, dtype=torch.float64, device=_DEV)
        for b, n in enumerate(s["lens"].tolist()):
            lo = max(0, n - case["window"]) if case["window"] else 0
            at = torch.arange(lo, n, device=_DEV)
            ids = s["table"][b].long()[at // page]
            for h in range(case["hkv"]):
                key = _exact_values(s["k"][ids, h, at % page], dim, s["k_scale"])
                score = key @ s["q"][b, h * g:(h + 1) * g].double().T * s["scale"]
                if case["softcap"]:
                    score = case["softcap"] * torch.tanh(score / case["softcap"])
                del key
                out[b, h * g:(h + 1) * g] = torch.softmax(score, 0).T @ _exact_values(s["v"][ids, h, at % page], dim, s["v_scale"])
        return out.reshape(case["batch"], -1)
    if kind in ("append", "read"):
        got = {}
        for name in ("k", "v"):
            out = torch.zeros(case["tokens"], case["hkv"], case["dim"], dtype=torch.float64, device=_DEV)
            has = s["slots"] >= 0
            slots = s["slots"][has]
            if kind == "append":
                out[has] = _exact_rounded(s["new_" + name][has], s[name + "_scale"])
            elif case["type"] == "e2m1":
                out[has] = _exact_values(s[name][slots // case["page"], :, slots % case["page"]], case["dim"], s[name + "_scale"])
            else:
                pool = s[name].float() if case["type"] == "e4m3" else s[name]
                out[has] = pool[slots // case["page"], :, slots % case["page"]].double() * s[name + "_scale"]
            got[name] = out
        return got
    probs = torch.zeros(case["rows"], dtype=torch.float64, device=_DEV)
    for i in range(case["rows"]):
        row, t = s["logits"][i].double(), float(s["temperature"][i])
        if t <= 0:
            probs[i] = 1.0
            continue
        p = torch.softmax(row / t, 0)
        # the tokens from the likeliest on (ties: the first one), and how many of them the options leave
        order = torch.sort(-row, stable=True).indices
        q = p[order]
        n, k = q.numel(), int(s["top_k"][i])
        n = min(n, k) if k > 0 else n
        top_p = float(s["top_p"][i])
        if top_p < 1:
            share = torch.cumsum(q[:n], 0) / q[:n].sum()
            n = min(n, int((share < top_p).sum()) + 1)
        n = max(1, min(n, int((q[:n] >= float(s["min_p"][i]) * q[0]).sum())))
        left = torch.zeros_like(p)
        left[order[:n]] = q[:n]
        run = torch.cumsum(left / left.sum(), 0)
        at = min(int(torch.searchsorted(run, float(s["uniforms"][i]), right=True)), run.numel() - 1)
        probs[i] = left[at] / left.sum()
    return {"tokens": None, "probs": probs}
