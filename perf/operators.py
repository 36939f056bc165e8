"""The operators of a decode step that serves many requests at once, and the work they are measured on.

Five operators: pages of a key-value cache handed to requests and taken back (`paged_reserve`, `paged_release`), key and
value rows written into their pages (`paged_append`), attention of one new token of each request over its pages
(`paged_attention`), and penalties, biases and grammar masks applied to the step's logits (`process_logits`).
`run` computes them in their plain form, in elementary torch operations, or with `own` by the backend's own calls.
"""
import math

import torch

own = False

_GOLDEN = 0.6180339887498949
_DTYPE = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "e4m3": torch.float8_e4m3fn}
_SIZE = {"f32": 4, "f16": 2, "bf16": 2, "e4m3": 1}
_DEV = "cuda"


# ---- the cases ---------------------------------------------------------------------------------------------------


def listed():
    return [
        # one short conversation on a sliding-window layer: the smallest call, where latency is all that counts
        dict(name="attend one", kind="attend", batch=1, max_len=333, hq=8, hkv=1, dim=256, page=16, type="bf16", window=512,
             softcap=0.0),
        # 64 conversations of every length up to 4096 on a full-attention layer with one key-value head: the ordinary step
        dict(name="attend batch", kind="attend", batch=64, max_len=4096, hq=8, hkv=1, dim=512, page=16, type="bf16", window=0,
             softcap=0.0),
        # a cache kept in 32 bits, several key-value heads, capped scores, an odd number of requests
        dict(name="attend f32 heads", kind="attend", batch=23, max_len=2501, hq=16, hkv=4, dim=128, page=32, type="f32", window=0,
             softcap=50.0),
        # three long documents in an 8-bit cache: few rows, so the length itself has to be split
        dict(name="attend long e4m3", kind="attend", batch=3, max_len=131072, hq=8, hkv=1, dim=512, page=64, type="e4m3", window=0,
             softcap=0.0),
        # the new token's key and value of 64 requests
        dict(name="append step", kind="append", tokens=64, hkv=1, dim=256, page=16, type="bf16"),
        # the rows of long prompts, rounded to 8 bits on their way into the pages
        dict(name="append prompts", kind="append", tokens=16411, hkv=1, dim=512, page=64, type="e4m3"),
        # one more token for each of 64 requests
        dict(name="reserve step", kind="reserve", batch=64, max_len=4096, max_new=1, page=16),
        # prompts of 512 new requests beside cached prefixes: about 131,000 tokens to place
        dict(name="reserve prompts", kind="reserve", batch=512, max_len=2000, max_new=512, page=16),
        # a few of 64 requests end, the others give back what a rejected draft had taken
        dict(name="release step", kind="release", batch=64, max_len=4096, page=16),
        # a full house of long requests gives back about half a million pages
        dict(name="release many", kind="release", batch=1031, max_len=16384, page=16),
        # one request's logits over a large vocabulary, a short history
        dict(name="logits one", kind="logits", rows=1, vocab=262144, history=900, bias=16, masks=1),
        # 64 requests with long histories, biases, and a grammar each of some of them
        dict(name="logits batch", kind="logits", rows=64, vocab=262144, history=8192, bias=300, masks=24),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["attend"] * 5 + ["append"] * 2 + ["reserve"] * 2 + ["release"] + ["logits"] * 2)
    page = rng.choice([16, 32, 64])
    if kind == "attend":
        dim, typ = rng.choice([64, 128, 256, 512]), rng.choice(["f32", "f16", "bf16", "bf16", "e4m3"])
        hkv, group = rng.choice([1, 1, 2, 4, 8]), rng.choice([1, 2, 4, 8, 8])
        row = 2 * hkv * dim * _SIZE[typ]
        rows = max(64, _log(rng, 2.0e5, 2.4e8) // row)  # tokens of all requests together
        batch = min(_log(rng, 1, 256), rows)
        return dict(kind=kind, batch=batch, max_len=min(131072, max(1, 2 * rows // batch - 1)), hq=hkv * group, hkv=hkv, dim=dim,
                    page=page, type=typ, window=rng.choice([0, 0, 512, 1000]), softcap=rng.choice([0.0, 0.0, 50.0]))
    if kind == "append":
        dim, hkv = rng.choice([64, 128, 256, 512]), rng.choice([1, 2, 4])
        return dict(kind=kind, tokens=_log(rng, 1, 16384 * 512 // (dim * hkv)), hkv=hkv, dim=dim, page=page,
                    type=rng.choice(["f32", "f16", "bf16", "e4m3"]))
    if kind == "reserve":
        batch = _log(rng, 1, 1024)
        return dict(kind=kind, batch=batch, max_len=_log(rng, 1, 4096), max_new=_log(rng, 1, max(1, 262144 // batch)), page=page)
    if kind == "release":
        batch = _log(rng, 1, 1024)
        return dict(kind=kind, batch=batch, max_len=_log(rng, 16, 16384), page=page)
    return dict(kind=kind, rows=_log(rng, 1, 64), vocab=_log(rng, 30000, 262144), history=_log(rng, 1, 8192),
                bias=rng.choice([0, 16, 300]), masks=rng.choice([0, 1, 8]))


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
        row = 2 * case["hkv"] * case["dim"] * _SIZE[case["type"]]
        pages = sum(_ceil(n, case["page"]) for n in keys)
        return {"bytes": sum(keys) * row + 8 * case["batch"] * case["hq"] * case["dim"] + 4 * pages + 4 * case["batch"],
                "flops": 4 * sum(keys) * case["hq"] * case["dim"]}
    if kind == "append":
        return {"bytes": case["tokens"] * (2 * case["hkv"] * case["dim"] * (4 + _SIZE[case["type"]]) + 8), "flops": 0}
    if kind == "reserve":
        lens, new = _spread(case["batch"], case["max_len"], 0), _spread(case["batch"], case["max_new"])[::-1]
        pages = sum(_ceil(a + b, case["page"]) - _ceil(a, case["page"]) for a, b in zip(lens, new))
        return {"bytes": 12 * case["batch"] + 8 * pages + 16 * sum(new) + 8, "flops": 0}
    if kind == "release":
        lens = _spread(case["batch"], case["max_len"])
        pages = sum(_ceil(n, case["page"]) - _ceil(k, case["page"]) for n, k in zip(lens, _kept(lens)))
        return {"bytes": 12 * case["batch"] + 8 * pages + 8, "flops": 0}
    hist = _spread(case["rows"], case["history"], 0)
    return {"bytes": case["rows"] * (8 * case["vocab"] + 24 + 8 * case["bias"]) + case["masks"] * _ceil(case["vocab"], 32) * 4
            + 4 * sum(hist), "flops": 2 * case["rows"] * case["vocab"]}


def _kept(lens):
    """What each request keeps: every third has ended, the others drop a rejected draft of up to 40 tokens."""
    return [0 if i % 3 == 0 else max(0, n - (7 * i) % 41) for i, n in enumerate(lens)]


# ---- what a program has in hand --------------------------------------------------------------------------------


def _ints(values, order=None):
    t = torch.tensor(values, dtype=torch.int32)
    return (t if order is None else t[order]).to(_DEV)


def _pages_of(lens, page, width, n_pages, gen):
    """A block table: every request's pages drawn at random from the pool, and the pages left over."""
    perm = torch.randperm(n_pages, generator=gen, device=_DEV).to(torch.int32)
    need = (lens.long() + page - 1) // page
    start = need.cumsum(0) - need
    col = torch.arange(width, device=_DEV)
    at = start[:, None] + col[None]
    table = torch.where(col[None] < need[:, None], perm[at.clamp(max=n_pages - 1)], torch.full_like(at, -1, dtype=torch.int32))
    return table.contiguous(), perm, int(need.sum())


def prepare(case, seed):
    gen = torch.Generator(device=_DEV)
    gen.manual_seed(int(seed))
    host = torch.Generator()
    host.manual_seed(int(seed))
    kind, s = case["kind"], {"kind": case["kind"], "case": case}
    if kind == "attend":
        batch, page, dim, hkv = case["batch"], case["page"], case["dim"], case["hkv"]
        lens = _ints(_spread(batch, case["max_len"]), torch.randperm(batch, generator=host))
        width = _ceil(case["max_len"], page)
        n_pages = int(sum(_ceil(n, page) for n in _spread(batch, case["max_len"]))) + 5
        table, _, _ = _pages_of(lens, page, width, n_pages, gen)
        # keys and values as they come out of their norms; the scale of an 8-bit cache leaves room for outliers
        scale = (1 / 32, 1 / 24) if case["type"] == "e4m3" else (1.0, 1.0)
        for name, sc in zip(("k", "v"), scale):
            pool = torch.empty(n_pages, hkv, page, dim, dtype=_DTYPE[case["type"]], device=_DEV)
            step = max(1, (64 << 20) // (hkv * page * dim))
            for i in range(0, n_pages, step):
                part = torch.randn(min(step, n_pages - i), hkv, page, dim, generator=gen, device=_DEV)
                pool[i:i + step] = (part / sc).clamp(-448, 448).to(pool.dtype) if case["type"] == "e4m3" else part.to(pool.dtype)
            s[name] = pool
        # what lies behind a request's last token is whatever the memory held: not a number here
        last, over = (lens.long() - 1) // page, (lens.long() - 1) % page + 1
        rows = torch.arange(page, device=_DEV)
        ids = table[torch.arange(batch, device=_DEV), last].long()
        stale = (rows[None] >= over[:, None])[:, None, :, None]
        for name in ("k", "v"):
            tail = s[name][ids].float()
            s[name][ids] = torch.where(stale, torch.full_like(tail, float("nan")), tail).to(s[name].dtype)
        s["q"] = 2.0 * torch.randn(batch, case["hq"], dim, generator=gen, device=_DEV)
        s["out"] = torch.empty(batch, case["hq"] * dim, device=_DEV)
        s.update(lens=lens, table=table, k_scale=scale[0], v_scale=scale[1], scale=dim ** -0.5, window=case["window"],
                 softcap=case["softcap"])
    elif kind == "append":
        n, page, dim, hkv = case["tokens"], case["page"], case["dim"], case["hkv"]
        n_pages = _ceil(n + n // 8, page) + 3
        s["new_k"] = torch.randn(n, hkv, dim, generator=gen, device=_DEV)
        s["new_v"] = torch.randn(n, hkv, dim, generator=gen, device=_DEV)
        slots = torch.randperm(n_pages * page, generator=gen, device=_DEV)[:n]
        slots[torch.arange(n, device=_DEV) % 97 == 96] = -1  # places of a padded batch: no row to write
        s["slots"] = slots
        for name in ("k", "v"):
            s[name] = torch.zeros(n_pages, hkv, page, dim, device=_DEV).to(_DTYPE[case["type"]])
        s["k_scale"], s["v_scale"] = (1 / 32, 1 / 24) if case["type"] == "e4m3" else (1.0, 1.0)
    elif kind == "reserve":
        batch, page = case["batch"], case["page"]
        order = torch.randperm(batch, generator=host)
        old, new = _spread(batch, case["max_len"], 0), _spread(batch, case["max_new"])[::-1]
        s["lens"], s["new"] = _ints(old, order), _ints(new, order)
        need = sum(_ceil(a + b, page) for a, b in zip(old, new))
        n_pages, s["width"] = need + 7, _ceil(case["max_len"] + case["max_new"], page)
        s["table"], perm, used = _pages_of(s["lens"], page, s["width"], n_pages, gen)
        s["free"] = torch.cat([perm[used:], torch.full((used,), -1, dtype=torch.int32, device=_DEV)])
        s["count"] = torch.tensor([n_pages - used], dtype=torch.int32, device=_DEV)
        tokens = sum(new) + 3  # a padded batch: the last places hold no token
        s["slots"] = torch.empty(tokens, dtype=torch.int64, device=_DEV)
        for name, n in (("positions", tokens), ("owners", tokens), ("totals", batch), ("left", 1)):
            s[name] = torch.empty(n, dtype=torch.int32, device=_DEV)
        s["page"] = page
    elif kind == "release":
        batch, page = case["batch"], case["page"]
        lens = _spread(batch, case["max_len"])
        order = torch.randperm(batch, generator=host)
        s["lens"], s["keep"] = _ints(lens, order), _ints(_kept(lens), order)
        used = sum(_ceil(n, page) for n in lens)
        n_pages, s["width"] = used + used // 4 + 5, _ceil(case["max_len"], page)
        s["table"], perm, _ = _pages_of(s["lens"], page, s["width"], n_pages, gen)
        s["free"] = torch.cat([perm[used:], torch.full((used,), -1, dtype=torch.int32, device=_DEV)])
        s["count"] = torch.tensor([n_pages - used], dtype=torch.int32, device=_DEV)
        s["totals"] = torch.empty(batch, dtype=torch.int32, device=_DEV)
        s["left"] = torch.empty(1, dtype=torch.int32, device=_DEV)
        s["page"] = page
    else:
        m, v, hist = case["rows"], case["vocab"], max(1, case["history"])
        s["logits"] = 4.0 * torch.randn(m, v, generator=gen, device=_DEV)
        # few tokens make up most of a text: the cube of a uniform number, spread over the vocabulary
        u = torch.rand(m, hist, generator=gen, device=_DEV) ** 3
        s["tokens"] = ((u * (v - 1)).long() * 7919 % v).to(torch.int32)
        lens = _ints(_spread(m, case["history"], 0), torch.randperm(m, generator=host))
        s["lens"], s["prompt"] = lens, (lens.float() * torch.rand(m, generator=gen, device=_DEV)).to(torch.int32)
        r = torch.rand(m, 3, generator=gen, device=_DEV)
        s["penalties"] = torch.stack([1.0 + 0.4 * r[:, 0], 0.8 * r[:, 1], 0.2 * r[:, 2]], 1).contiguous()
        n = case["bias"]
        first = torch.randint(0, v, (m, 1), generator=gen, device=_DEV)
        s["bias_ids"] = ((first + torch.arange(n, device=_DEV)[None] * (v // max(1, n))) % v).to(torch.int32).reshape(-1)
        s["bias_values"] = 10.0 * torch.rand(m * n, generator=gen, device=_DEV) - 5.0
        s["bias_offsets"] = (torch.arange(m + 1, device=_DEV) * n).to(torch.int32)
        words, k = _ceil(v, 32), case["masks"]
        bits = torch.randint(-2 ** 31, 2 ** 31, (3, k, words), generator=gen, device=_DEV)
        s["masks"] = (bits[0] & bits[1] & bits[2]).to(torch.int32)
        s["mask_rows"] = torch.where(torch.arange(m, device=_DEV) < k, torch.arange(m, device=_DEV), -1).to(torch.int32)
        s["out"] = torch.empty(m, v, device=_DEV)
    return s


# ---- the plain forms ---------------------------------------------------------------------------------------------


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
    keys = (k[ids].float() * s["k_scale"]).transpose(1, 2).reshape(batch, hkv, -1, dim)
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
    values = (v[ids].float() * s["v_scale"]).transpose(1, 2).reshape(batch, hkv, -1, dim)
    values = torch.where(row, values, torch.zeros_like(values))
    out = torch.matmul(p, values) / torch.where(total == 0, torch.ones_like(total), total)
    return out.reshape(batch, hq * dim)


def _append_plain(s):
    page = s["k"].shape[2]
    take = (s["slots"] >= 0).nonzero().squeeze(1)
    slots = s["slots"][take]
    for pool, rows, scale in ((s["k"], s["new_k"], s["k_scale"]), (s["v"], s["new_v"], s["v_scale"])):
        x = rows[take]
        if pool.dtype == torch.float8_e4m3fn:
            x = (x * (1.0 / scale)).clamp(-448, 448).to(pool.dtype)
            pool.view(torch.uint8)[slots // page, :, slots % page] = x.view(torch.uint8)
        else:
            pool[slots // page, :, slots % page] = x.to(pool.dtype)
    return {"k": s["k"], "v": s["v"]}


def _reserve_plain(s):
    page, table, free = s["page"], s["table"], s["free"]
    old, new = s["lens"].long().clamp(min=0), s["new"].long().clamp(min=0)
    had, have = (old + page - 1) // page, (old + new + page - 1) // page
    need, ends = have - had, new.cumsum(0)
    first = need.cumsum(0) - need
    count = s["count"].long()
    fits = (need.sum() <= count) & (have.max() <= s["width"]) & (ends[-1] <= s["slots"].numel())
    col = torch.arange(s["width"], device=free.device)
    taken = (col[None] >= had[:, None]) & (col[None] < have[:, None]) & fits
    pick = (count - 1 - (first[:, None] + col[None] - had[:, None])).clamp(0, free.numel() - 1)
    table.copy_(torch.where(taken, free[pick], table))
    t = torch.arange(s["slots"].numel(), device=free.device)
    owner = torch.searchsorted(ends, t, right=True).clamp(max=old.numel() - 1)
    real = (t < ends[-1]) & fits
    pos = old[owner] + t - (ends - new)[owner]
    slot = table[owner, (pos // page).clamp(0, s["width"] - 1)].long() * page + pos % page
    return {"table": table, "slots": torch.where(real, slot, -1),
            "positions": torch.where(real, pos, 0).to(torch.int32), "owners": torch.where(real, owner, -1).to(torch.int32),
            "totals": torch.where(fits, old + new, old).to(torch.int32), "left": torch.where(fits, count - need.sum(), count).to(torch.int32)}


def _release_plain(s):
    page, free = s["page"], s["free"]
    old = s["lens"].long().clamp(min=0)
    keep = torch.minimum(s["keep"].long().clamp(min=0), old)
    had, have = (old + page - 1) // page, (keep + page - 1) // page
    back = had - have
    first, count = back.cumsum(0) - back, s["count"].long()
    total = back.sum()
    fits = count + total <= free.numel()
    col = torch.arange(s["width"], device=free.device)
    given = (col[None] >= have[:, None]) & (col[None] < had[:, None]) & fits
    to = count + total - 1 - (first[:, None] + col[None] - have[:, None])
    to = torch.where(given, to, free.numel())
    more = torch.cat([free, free.new_zeros(1)])
    more[to.reshape(-1)] = s["table"].reshape(-1)
    free.copy_(more[:-1])
    return {"free": free, "left": torch.where(fits, count + total, count).to(torch.int32),
            "totals": torch.where(fits, keep, old).to(torch.int32)}


def _logits_plain(s):
    l = s["logits"]
    m, v = l.shape
    tok, at = s["tokens"].long(), torch.arange(s["tokens"].shape[1], device=l.device)[None]
    valid = (at < s["lens"].long()[:, None]) & (tok >= 0) & (tok < v)
    made = valid & (at >= s["prompt"].long()[:, None])
    seen = torch.zeros(m, v + 1, device=l.device).scatter_(1, torch.where(valid, tok, v), 1.0)[:, :v] > 0
    count = torch.zeros(m, v + 1, device=l.device).scatter_add_(1, torch.where(made, tok, v), made.float())[:, :v]
    rep, presence, frequency = (c[:, None] for c in s["penalties"].unbind(1))
    l = torch.where(seen, torch.where(l > 0, l / rep, l * rep), l)
    l = l - frequency * count
    l = l - presence * (count > 0)
    n = s["bias_ids"].numel()
    row = torch.searchsorted(s["bias_offsets"].long(), torch.arange(n, device=l.device), right=True) - 1
    bias = torch.zeros(m, v, device=l.device)
    bias[row, s["bias_ids"].long()] = s["bias_values"]
    l = l + bias
    if s["masks"].shape[0]:
        bits = (s["masks"][:, :, None] >> torch.arange(32, dtype=torch.int32, device=l.device)) & 1
        allowed = bits.reshape(s["masks"].shape[0], -1)[:, :v] == 1
        of = s["mask_rows"].long()
        l = torch.where(allowed[of.clamp(min=0)] | (of < 0)[:, None], l, torch.full_like(l, -math.inf))
    return l


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
    if kind == "append":
        g.paged_append(_pages(s), s["new_k"], s["new_v"], s["slots"])
        return {"k": s["k"], "v": s["v"]}
    if kind == "reserve":
        g.paged_reserve(s["lens"], s["new"], s["page"], s["table"], s["free"], s["count"], slots=s["slots"],
                        positions=s["positions"], owners=s["owners"], totals=s["totals"], free_left=s["left"])
        return {k: s[k] for k in ("table", "slots", "positions", "owners", "totals", "left")}
    if kind == "release":
        g.paged_release(s["lens"], s["keep"], s["page"], s["table"], s["free"], s["count"], totals=s["totals"], free_left=s["left"])
        return {k: s[k] for k in ("free", "left", "totals")}
    g.process_logits(s["logits"], tokens=s["tokens"], prompt_lens=s["prompt"], lens=s["lens"], penalties=s["penalties"],
                     bias_ids=s["bias_ids"], bias_values=s["bias_values"], bias_offsets=s["bias_offsets"], masks=s["masks"],
                     mask_rows=s["mask_rows"], out=s["out"])
    return s["out"]


_PLAIN = {"attend": _attend_plain, "append": _append_plain, "reserve": _reserve_plain, "release": _release_plain,
          "logits": _logits_plain}


def run(state):
    return _run_own(state) if own else _PLAIN[state["kind"]](state)


# ---- the definitions, in 64 bits ---------------------------------------------------------------------------------


def exact(case, seed):
    kind = case["kind"]
    if kind in ("reserve", "release"):
        return None  # whole numbers
    s = prepare(case, seed)
    if kind == "attend":
        page, dim, g = case["page"], case["dim"], case["hq"] // case["hkv"]
        out = torch.zeros(case["batch"], case["hq"], dim, dtype=torch.float64, device=_DEV)
        for b, n in enumerate(s["lens"].tolist()):
            lo = max(0, n - case["window"]) if case["window"] else 0
            at = torch.arange(lo, n, device=_DEV)
            ids = s["table"][b].long()[at // page]
            for h in range(case["hkv"]):
                key = s["k"][ids, h, at % page].double() * s["k_scale"]
                score = key @ s["q"][b, h * g:(h + 1) * g].double().T * s["scale"]
                if case["softcap"]:
                    score = case["softcap"] * torch.tanh(score / case["softcap"])
                out[b, h * g:(h + 1) * g] = torch.softmax(score, 0).T @ (s["v"][ids, h, at % page].double() * s["v_scale"])
        return out.reshape(case["batch"], -1)
    if kind == "append":
        pools = {}
        for name in ("k", "v"):
            flat = torch.zeros(s[name].numel() // (case["hkv"] * case["dim"]), case["hkv"], case["dim"], dtype=torch.float64, device=_DEV)
            rows = s["slots"] >= 0
            x = s["new_" + name].double() / (s[name + "_scale"])
            if case["type"] == "e4m3":
                # the nearest number of 4 exponent and 3 fraction bits, ties to even; the largest is 448
                exp = torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6)))
                x = (torch.round(x / 2.0 ** (exp - 3)) * 2.0 ** (exp - 3)).clamp(-448, 448)
            flat[s["slots"][rows]] = x[rows]
            pools[name] = flat.view(-1, case["page"], case["hkv"], case["dim"]).transpose(1, 2).contiguous()
        return pools
    m, v = case["rows"], case["vocab"]
    out = s["logits"].double()
    offsets = s["bias_offsets"].tolist()
    for i, (n, p) in enumerate(zip(s["lens"].tolist(), s["prompt"].tolist())):
        rep, presence, frequency = s["penalties"][i].double().tolist()
        tok = s["tokens"][i].long()
        was = tok[:n].unique()
        row = out[i]
        row[was] = torch.where(row[was] > 0, row[was] / rep, row[was] * rep)
        made = torch.bincount(tok[p:n], minlength=v).double()
        row -= frequency * made + presence * (made > 0)
        a, b = offsets[i], offsets[i + 1]
        row[s["bias_ids"][a:b].long()] += s["bias_values"][a:b].double()
        mask = int(s["mask_rows"][i])
        if mask >= 0:
            col = torch.arange(v, device=_DEV)
            row[(s["masks"][mask][col // 32] >> (col % 32)) & 1 == 0] = -math.inf
    return out
