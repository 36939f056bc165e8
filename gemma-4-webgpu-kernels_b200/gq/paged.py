"""Decoding many requests of different lengths at once, over a paged KV cache.

``PagedDecoder`` is the decode step of ``gq.e2b`` with the cache in pages: each of its
``batch`` places holds a request with a length of its own, and a step

* takes pages for the new tokens (``gq_paged_reserve``: positions and slots of the step,
  brought to their places, since places without a request get none),
* writes each KV layer's new rows into their pages (``gq_paged_append``),
* attends every request over its own pages (``gq_paged_attention``),
* applies each request's penalties, biases and grammar mask to its logits
  (``gq_process_logits``) and samples (``gq_sample_rows``),
* takes back the pages of requests that have ended (``gq_paged_release``).

Lengths, tables, free pages, histories and controls live on the device, so one recorded
graph serves every step. No counterpart in the reference (one sequence, contiguous
caches).

    python -m gq.paged [--requests 64] [--steps 32] [--type bf16]

decodes with synthetic E2B-shaped weights and prints the time of a step.
"""
from __future__ import annotations

import argparse
import ctypes
import sys
from contextlib import contextmanager
from ctypes import c_float, c_void_p
from typing import Optional, Sequence

import numpy as np

from . import _abi, e2b
from ._abi import GqError

KEEP_ALL = 2 ** 31 - 1


class PagedDecoder(e2b.Decoder):
    """One decode step of ``batch`` requests through the C ABI, over pages.

    max_len: the most tokens of a request (its block table row); page_size, kv_type
    ("f32", "f16", "bf16", "e4m3" with k_scale / v_scale) and n_pages (default: enough
    for every request at max_len) describe the pool that each source layer has. ``lens``
    are the requests' lengths, filled by ``extend``. A place whose request has ended idles,
    and a request of max_len tokens stands still: a step takes no page for them, leaves
    their token as it is, and their rows of the logits mean nothing.

    Controls, all device tensors that may be changed between steps on torch's current
    stream (whatever stream the backend has, a step comes after what that stream was given
    before it, and the stream goes on after the step): ``penalties`` [batch, 3]
    (repetition, presence, frequency), ``prompt_lens`` [batch], ``history`` [batch,
    max_len] (tokens by position, -1 where they are not known), and, given at construction
    because their sizes belong to the recorded step, ``bias`` (ids, values, offsets) and
    ``masks`` (words, rows); see gq_process_logits in include/gq.h. ``sample``: temperature,
    top_k, top_p of gq_sample_rows."""

    def __init__(self, g, cfg: e2b.Config, weights: Optional[e2b.Weights], batch: int, max_len: int, page_size: int = 16,
                 kv_type: str = "bf16", n_pages: Optional[int] = None, k_scale: float = 1.0, v_scale: float = 1.0,
                 sample=(0.0, 0, 1.0), bias=None, masks=None, seed: int = 1, device_init_seed: Optional[int] = None):
        self.page_size, self.kv_type, self.width = page_size, kv_type, -(-max_len // page_size)
        self.n_pages = n_pages if n_pages is not None else batch * self.width
        self.k_scale, self.v_scale = k_scale, v_scale
        self.bias, self.masks = bias, masks
        self.opts = _abi.SampleOpts(float(sample[0]), int(sample[1]), float(sample[2]), 1.0)
        self.seed = seed
        super().__init__(g, cfg, weights, batch, cache_len=0, capacity=max_len, device_init_seed=device_init_seed,
                         fuse_norms=False)
        self.graph = None
        self.torch.cuda.synchronize(g.torch_device)

    # ---- the cache -------------------------------------------------------------------
    def _make_kv(self, weights, kv_gen, kv_device_seed) -> None:
        torch, c, g, B = self.torch, self.cfg, self.g, self.batch
        dev, i32 = g.torch_device, torch.int32
        dtypes = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "e4m3": torch.float8_e4m3fn}
        if self.kv_type not in dtypes:
            raise GqError(_abi.GQ_ERR_UNSUPPORTED, f"PagedDecoder: kv_type {self.kv_type}")
        self.kcache, self.vcache, self.pages = {}, {}, {}
        for i in range(c.layers):
            if c.kv_source(i) == i:
                shape = (self.n_pages, c.heads_kv, self.page_size, c.dh(i))
                k, v = (torch.empty(shape, dtype=dtypes[self.kv_type], device=dev) for _ in range(2))
                self.pages[i] = g.kv_pages(k, v, self.k_scale, self.v_scale)
        self.table = torch.full((B, max(self.width, 1)), -1, dtype=i32, device=dev)
        self.free = torch.arange(self.n_pages, dtype=i32, device=dev)
        self.count = torch.tensor([self.n_pages], dtype=i32, device=dev)
        self.lens = torch.zeros(B, dtype=i32, device=dev)
        self.now = torch.zeros(B, dtype=i32, device=dev)  # the lengths with the step's tokens
        self.took = torch.zeros(B, dtype=torch.bool, device=dev)
        self.keep = torch.full((B,), KEEP_ALL, dtype=i32, device=dev)
        # a place below its limit takes a token: max_len, and 0 where no request is
        self.limit = torch.full((B,), self.capacity, dtype=i32, device=dev)
        self.new = torch.zeros(B, dtype=i32, device=dev)
        self.ending = set()  # places that were ended and whose last step is still to come
        # the step's tokens in the order of gq_paged_reserve, which leaves out places without
        # one, and then by place (one more: what is left over goes there)
        self.slots = torch.zeros(B, dtype=torch.int64, device=dev)
        self.positions = torch.zeros(B, dtype=i32, device=dev)
        self.owners = torch.zeros(B, dtype=i32, device=dev)
        self.place = torch.zeros(B, dtype=torch.int64, device=dev)
        self.place_slots = torch.full((B + 1,), -1, dtype=torch.int64, device=dev)
        self.place_pos = torch.zeros(B + 1, dtype=i32, device=dev)
        d = c.heads_kv * c.global_head_dim
        self.new_k, self.new_v = (torch.zeros(B, max(d, c.heads_kv * c.head_dim), device=dev) for _ in range(2))
        # controls of the logits
        # (a column more: a request that stands still at max_len puts its id there)
        self.ids_at = torch.zeros(B, self.capacity + 1, dtype=i32, device=dev)
        self.history = self.ids_at[:, :self.capacity]
        self.prompt_lens = torch.zeros(B, dtype=i32, device=dev)
        self.penalties = torch.tensor([[1.0, 0.0, 0.0]], device=dev).repeat(B, 1)
        self.controlled = torch.empty(B, c.vocab, device=dev)
        self.tokens = torch.zeros(B, dtype=i32, device=dev)
        self.rng = torch.arange(self.seed, self.seed + B, dtype=torch.int64, device=dev)
        self.drawn, self.rng_after = torch.zeros_like(self.tokens), torch.zeros_like(self.rng)  # of the step
        torch.cuda.synchronize(dev)

    def _stream(self):
        return self.torch.cuda.ExternalStream(self.g.stream_ptr(), device=self.g.torch_device)

    @contextmanager
    def _ordered(self):
        """Work on the backend's stream that comes after what torch's current stream was given
        so far, and before what it is given next."""
        mine, callers = self._stream(), self.torch.cuda.current_stream(self.g.torch_device)
        apart = (callers.cuda_stream or 1) != mine.cuda_stream  # (1: the legacy default stream, as the backend has it)
        if apart:
            mine.wait_stream(callers)
        try:
            with self.torch.cuda.stream(mine):
                yield
        finally:
            if apart:
                callers.wait_stream(mine)

    def extend(self, new_lens: Sequence[int], rows, tokens: Optional[Sequence[Sequence[int]]] = None) -> None:
        """Add new_lens[b] tokens to request b without decoding (a prompt's cache made
        elsewhere): rows(layer) gives their keys and values, f32 [sum, heads_kv *
        head_dim] in request order, for each source layer; tokens, when given, each
        request's ids, as many as are known (its prompt, for the penalties; all that an
        extended request holds counts as its prompt from then on). A place whose request
        was ended begins anew, whether a step has come between or not. Raises when the
        pages do not suffice, when a request would pass max_len, and what earlier steps
        left to raise; no page is taken then."""
        torch, c, g = self.torch, self.cfg, self.g
        new_lens = [int(n) for n in new_lens]
        if len(new_lens) != self.batch or min(new_lens) < 0:
            raise GqError(_abi.GQ_ERR_INVALID_ARGUMENT, f"extend: new_lens must be {self.batch} lengths")
        if tokens is not None and (len(tokens) > self.batch or any(len(ids) > n for ids, n in zip(tokens, new_lens))):
            raise GqError(_abi.GQ_ERR_INVALID_ARGUMENT, "extend: more ids than new tokens")
        dev, total = g.torch_device, sum(new_lens)
        place = lambda dt: torch.empty(total, dtype=dt, device=dev)  # noqa: E731
        g.flush()  # steps in flight change the lengths; their errors are raised before anything is taken
        new, slots = torch.tensor(new_lens, dtype=torch.int32, device=dev), place(torch.int64)
        anew = (new > 0) & (self.keep == 0)  # places whose end no step has carried out yet: it is now
        if bool((torch.where(anew, 0, self.lens) + new > self.capacity).any()):
            raise GqError(_abi.GQ_ERR_INVALID_ARGUMENT, f"extend: a request would hold more than {self.capacity} tokens")
        if bool(anew.any()):
            keep = torch.where(anew, 0, KEEP_ALL).to(torch.int32)
            torch.cuda.synchronize(dev)
            g.paged_release(self.lens, keep, self.page_size, self.table, self.free, self.count, self.lens, self.count)
            g.flush()
            # (whatever becomes of what follows, the place is idle now)
            self.limit.masked_fill_(anew, 0)
            self.ending -= {b for b, n in enumerate(new_lens) if n > 0}
        before = self.lens.tolist()
        pos, owners = place(torch.int32), place(torch.int32)
        kv = {i: rows(i) for i in self.pages} if total else {}
        torch.cuda.synchronize(dev)  # (the rows are torch's, the calls go to the backend's stream)
        g.paged_reserve(self.lens, new, self.page_size, self.table, self.free, self.count, slots, pos, owners, self.lens,
                        self.count)
        g.flush()
        for i, (k, v) in kv.items():
            g.paged_append(self.pages[i], k.view(total, c.heads_kv, c.dh(i)), v.view(total, c.heads_kv, c.dh(i)), slots)
        g.flush()
        # ids that are not given are -1, which the penalties ignore
        at, first = torch.arange(self.capacity, device=dev)[None], torch.tensor(before, device=dev)[:, None]
        self.history.masked_fill_((at >= first) & (at < first + new[:, None]), -1)
        if tokens is not None:
            for b, ids in enumerate(tokens):
                self.history[b, before[b]:before[b] + len(ids)] = torch.tensor(list(ids), dtype=torch.int32, device=dev)
        # (requests that were not extended keep theirs: what they generated stays generated)
        self.prompt_lens.copy_(torch.where(new > 0, self.lens, self.prompt_lens))
        self.keep.masked_fill_(new > 0, KEEP_ALL)
        self.limit.masked_fill_(new > 0, self.capacity)
        self.ending -= {b for b, n in enumerate(new_lens) if n > 0}
        torch.cuda.synchronize(dev)

    def end(self, places: Sequence[int]) -> None:
        """The requests at these places end: the next step is their last, and gives their pages
        back. The places idle from then on, until ``extend`` gives them a request."""
        places = [int(b) for b in places]
        if any(not 0 <= b < self.batch for b in places):  # (on the device an index past the end is a fault)
            raise GqError(_abi.GQ_ERR_INVALID_ARGUMENT, f"end: places are 0 to {self.batch - 1}")
        with self._ordered():
            self.keep[self.torch.tensor(places, dtype=self.torch.int64, device=self.g.torch_device)] = 0
        self.ending |= set(places)

    # ---- the step ----------------------------------------------------------------------
    def set_position(self, p: int) -> None:
        """(Every request has its own position; the calls are the same for every step.)"""
        self.pos = self.place_pos[:self.batch]
        self._calls = self._build_calls(0)

    def _begin_calls(self, add) -> None:
        V = lambda t: c_void_p(t.data_ptr())  # noqa: E731
        add("new", self._torch_call, lambda: self.torch.gt(self.limit, self.lens, out=self.new))
        add("reserve", self.g.lib.gq_paged_reserve, self.g.ctx, self.batch, self.page_size, V(self.lens), V(self.new),
            V(self.table), self.table.shape[1], V(self.free), self.n_pages, V(self.count), V(self.count), self.batch,
            V(self.slots), V(self.positions), V(self.owners), V(self.now))
        add("place", self._torch_call, self._place_tokens)

    def _place_tokens(self) -> None:
        """Slots and positions by place: -1 (no row is written) and any position where the step
        has no token of the place."""
        self.torch.remainder(self.owners, self.batch + 1, out=self.place)  # (no owner, -1: the place past the last)
        self.place_slots.fill_(-1)
        self.place_slots.scatter_(0, self.place, self.slots)
        self.place_pos.scatter_(0, self.place, self.positions)

    def _new_rows(self, src: int, p: int, kvd: int):
        return c_void_p(self.new_k.data_ptr()), c_void_p(self.new_v.data_ptr()), kvd

    def _attention_calls(self, add, pre: str, i: int, src: int, dh: int, p: int) -> None:
        c, V, lib, ctx = self.cfg, lambda t: c_void_p(t.data_ptr()), self.g.lib, self.g.ctx  # noqa: E731
        pages = c_void_p(self.pages[src].ref)
        if src == i:
            add(pre + "append", lib.gq_paged_append, ctx, pages, V(self.new_k), V(self.new_v), self.batch, 0, 0,
                V(self.place_slots))
        add(pre + "attention", lib.gq_paged_attention, ctx, pages, V(self.qr), self.batch, c.heads_q, 0, V(self.table),
            self.table.shape[1], V(self.now), c_float(1.0), c.window_of(i), c_float(0.0), V(self.attn))

    def _end_calls(self, add) -> None:
        V = lambda t: c_void_p(t.data_ptr())  # noqa: E731
        lib, ctx, B, vocab = self.g.lib, self.g.ctx, self.batch, self.cfg.vocab
        d, i32, n_bias, n_masks, mask_words = self.g._dev, self.torch.int32, 0, 0, 0
        ids = values = offsets = words = rows = None
        if self.bias is not None:
            n_bias = self.bias[0].numel()
            ids, offsets = d(self.bias[0], i32, "bias: ids"), d(self.bias[2], i32, "bias: offsets", B + 1)
            values = d(self.bias[1], self.torch.float32, "bias: values", n_bias)
        if self.masks is not None:
            if self.masks[0].dim() != 2:
                raise GqError(_abi.GQ_ERR_INVALID_ARGUMENT, "masks: words must be [k, words]")
            words, (n_masks, mask_words) = d(self.masks[0], i32, "masks: words"), self.masks[0].shape
            if mask_words < -(-vocab // 32) or (self.masks[1] is None and n_masks < B):
                raise GqError(_abi.GQ_ERR_INVALID_ARGUMENT, "masks: too few words of a row, or rows")
            rows = d(self.masks[1], i32, "masks: rows", B) if self.masks[1] is not None else None
        add("process_logits", lib.gq_process_logits_bounded, ctx, V(self.logits), B, vocab, vocab, V(self.ids_at),
            self.capacity + 1, V(self.prompt_lens), V(self.now), V(self.penalties), ids, values, offsets, n_bias, words,
            n_masks, mask_words, rows, V(self.controlled), vocab)
        if self.opts.temperature > 0:
            add("rng", self._torch_call, lambda: self.rng_after.copy_(self.rng))
        add("sample", lib.gq_sample_rows, ctx, V(self.controlled), B, vocab, vocab, ctypes.byref(self.opts), None, 0, 0,
            V(self.rng_after), V(self.drawn))
        add("keep", self._torch_call, self._take_tokens)
        add("release", lib.gq_paged_release, ctx, B, self.page_size, V(self.now), V(self.keep), V(self.table),
            self.table.shape[1], V(self.free), self.n_pages, V(self.count), V(self.count), V(self.lens))

    def _torch_call(self, fn) -> int:
        """One of the step's calls that is torch's: on the backend's stream, into tensors that
        are there already (the step is recorded)."""
        with self.torch.cuda.stream(self._stream()):
            fn()
        return _abi.GQ_OK

    def _take_tokens(self) -> None:
        """The drawn tokens become the requests', except where the step placed no token."""
        torch = self.torch
        torch.ne(self.now, self.lens, out=self.took)
        torch.where(self.took, self.drawn, self.tokens, out=self.tokens)
        if self.opts.temperature > 0:  # (a greedy step draws no numbers)
            torch.where(self.took, self.rng_after, self.rng, out=self.rng)

    def step(self, ids=None):
        """Decode one token of every request (of less than max_len tokens): ids [batch] (default: the tokens that the last
        step sampled) in, the sampled ``tokens`` [batch] out (a device tensor, valid until
        the next step). Enqueued; a page shortage shows at the next ``g.flush()``: the step
        then decoded nothing. Lengths, tokens and random states are as they were, and only
        the pages of requests that were ended have gone back, so that it can be repeated.
        ``took`` [batch] tells which requests the last step has decoded a token of."""
        torch = self.torch
        with self._ordered():
            if ids is None:
                self.ids.copy_(self.tokens)
            else:
                self.ids.copy_(torch.as_tensor(np.asarray(ids, dtype=np.int32).reshape(self.batch)))
            self.ids_at.scatter_(1, self.lens.long()[:, None], self.ids[:, None])
            if self.graph is not None:
                self.g.replay(self.graph)
            else:
                self.run()
            if self.ending:
                self.limit[torch.tensor(sorted(self.ending), device=self.g.torch_device)] = 0
                self.ending.clear()
        return self.tokens

    def record_steps(self) -> None:
        """Record the step into a graph that ``step`` replays from now on (the backend must
        own its stream). Runs one step first, which sizes the workspaces, and takes its
        token back: lengths, pages and random states are as before."""
        torch = self.torch
        self.g.flush()
        saved = [(t, t.clone()) for t in (self.lens, self.table, self.free, self.count, self.rng, self.tokens, self.took)]
        torch.cuda.synchronize(self.g.torch_device)
        try:
            self.run()
            self.g.flush()
        finally:
            for t, old in saved:
                t.copy_(old)
            torch.cuda.synchronize(self.g.torch_device)
        self.graph = self.g.record(self.run)

    def close(self) -> None:
        if self.graph is not None:
            self.g.destroy_graph(self.graph)
            self.graph = None
        super().close()
        self.pages.clear()

    def kv_bytes(self) -> int:
        """K and V bytes that a step's attention reads at the present lengths."""
        c, size = self.cfg, {"f32": 4, "e4m3": 1}.get(self.kv_type, 2)
        self._stream().synchronize()
        lens, tot = self.lens.tolist(), 0
        for i in range(c.layers):
            w = c.window_of(i)
            tot += 2 * sum(min(n, w) if w else n for n in lens) * c.heads_kv * c.dh(i) * size
        return tot


def main(argv=None) -> int:
    ap = argparse.ArgumentParser(prog="gq.paged")
    ap.add_argument("--requests", type=int, default=64)
    ap.add_argument("--max-len", type=int, default=2048)
    ap.add_argument("--steps", type=int, default=32)
    ap.add_argument("--type", choices=["f32", "f16", "bf16", "e4m3"], default="bf16")
    args = ap.parse_args(argv)

    import torch

    from . import CudaBackend

    g = CudaBackend(0, own_stream=True)
    cfg, B = e2b.e2b_config(), args.requests
    scales = dict(k_scale=1 / 32, v_scale=1 / 32) if args.type == "e4m3" else {}
    dec = PagedDecoder(g, cfg, None, B, args.max_len, kv_type=args.type, sample=(1.0, 64, 0.95), device_init_seed=5, **scales)
    gen = torch.Generator(device=g.torch_device)
    gen.manual_seed(6)
    room = max(1, args.max_len - args.steps - 4)
    lens = np.random.default_rng(7).integers(1, room + 1, B)
    total = int(lens.sum())

    def rows(layer):
        return [torch.randn(total, cfg.heads_kv * cfg.dh(layer), generator=gen, device=g.torch_device) for _ in range(2)]

    dec.extend(lens, rows)
    dec.penalties.copy_(torch.tensor([[1.1, 0.2, 0.1]], device=g.torch_device))
    dec.record_steps()
    dec.step(np.arange(B) % cfg.vocab)
    g.flush()
    t0, t1 = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    t0.record(dec._stream())
    for _ in range(args.steps):
        dec.step()
    t1.record(dec._stream())
    g.flush()
    ms = t0.elapsed_time(t1) / args.steps
    print(f"{B} requests of 1 to {room} tokens ({args.type} pages): {ms:.3f} ms per step, {B / ms * 1e3:.0f} tokens/s, "
          f"{dec.kv_bytes() / 1e6:.0f} MB of keys and values read per step")
    dec.close()
    g.close()
    return 0


if __name__ == "__main__":
    sys.exit(main())
