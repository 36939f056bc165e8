"""gq — B200 backend for the quantized-weight hot path of the Gemma-4 engine.

Host-side mirror of the reference's `Backend` trait (rust/src/backend.rs:88-180)
for the quantized ops, on top of the C ABI in include/gq.h (libgq.so). Method
names, argument meaning and error behaviour follow the trait:

* ``quant_tensor(QuantWeight)``                        rust/src/backend.rs:95
* ``linear(x, w)``                                     rust/src/backend.rs:105-106
* ``linear_geglu(x, w_gate, w_up)``                    rust/src/backend.rs:155-160
* ``linear_gelu_mul_cols(x, w, b, offset)``            rust/src/backend.rs:161-167
* ``embed_rows(table, ids, scale)``                    rust/src/backend.rs:101-102
* ``softcap(a, cap)`` / ``geglu(gate, up)``            rust/src/backend.rs:113-116
* ``tensor`` / ``zeros`` / ``reshape`` / ``readback`` / ``flush`` /
  ``begin_frame`` / ``end_frame`` / ``free_tensor``    rust/src/backend.rs:94-98, 169-179
* support ops of a decode step: ``rms_norm``, ``add``, ``mul``, ``scale``,
  ``scale_by_tensor``, ``rope``, ``attention``, ``slice_rows``, ``slice_cols``,
  ``concat_rows``, ``kv_append`` (rust/src/backend.rs:103-130), ``add_rms_norm``,
  ``head_norm_rope`` (:137-154), and ``linear`` with a bf16-stored plain weight
* the paged cache and the logits of a step that serves many requests (no counterpart in
  the trait): ``kv_pages``, ``paged_reserve``, ``paged_release``, ``paged_append``,
  ``paged_read``, ``paged_attention``, ``process_logits``, ``sample_requests``

Ops enqueue on the backend's stream (torch's current stream of the device) and
return immediately; ``readback`` blocks, like the reference. Failures raise
``GqError`` where the Rust trait panics. Device memory for f32 tensors comes from
torch's caching allocator; the quantized weights are owned by libgq.
"""
from __future__ import annotations

import ctypes
from ctypes import c_float, c_int32, c_int64, c_uint8, c_void_p
from dataclasses import dataclass, field
from typing import Optional, Sequence

import numpy as np

from . import _abi
from ._abi import GqError

__all__ = ["QuantWeight", "GqTensor", "CudaBackend", "GqError", "AttnOpts", "KvAppend", "KvPages"]


@dataclass
class QuantWeight:
    """A weight kept in its packed, quantized form (rust/src/backend.rs:16-24).

    ``qbytes``: raw payload (U8 sub-byte packed LSB-first offset-binary, or
    native I8); ``scales``: one f32 per (row, group); ``shape``: logical [N, K].
    """

    qbytes: np.ndarray
    scales: np.ndarray
    shape: tuple
    bits: int
    signed_i8: bool
    group_size: int

    def per_byte(self) -> int:  # rust/src/backend.rs:28-30
        return 1 if self.signed_i8 else 8 // self.bits

    def row_bytes(self) -> int:  # rust/src/backend.rs:33-36
        k = self.shape[1]
        return k if self.signed_i8 else k // self.per_byte()

    def scale_stride(self) -> int:  # rust/src/backend.rs:39-41
        return -(-self.shape[1] // self.group_size)

    def codes(self) -> np.ndarray:
        """All integer codes [N, K] (the integer part of deq, backend.rs:46-54)."""
        n, k = self.shape
        b = np.asarray(self.qbytes, dtype=np.uint8)[: n * self.row_bytes()].reshape(n, self.row_bytes())
        if self.signed_i8:
            return b.view(np.int8).astype(np.int32)
        pb = self.per_byte()
        shifts = (np.arange(pb, dtype=np.uint32) * self.bits)[None, None, :]
        raw = (b.astype(np.uint32)[:, :, None] >> shifts) & ((1 << self.bits) - 1)
        return raw.reshape(n, k).astype(np.int32) - (1 << (self.bits - 1))


@dataclass
class GqTensor:
    """A backend tensor: dense row-major f32 on the device, a quantized weight, or a
    plain weight stored as bf16 (``bf16=True``: ``data`` is a cuda int16 tensor of
    the bf16 bit patterns)."""

    shape: tuple
    data: object = None          # torch.Tensor (cuda, float32, contiguous) for f32 tensors
    qw: Optional[int] = None     # gq_qweight* for quantized tensors
    quant: Optional[QuantWeight] = field(default=None, repr=False)
    bf16: bool = False

    def size(self) -> int:
        return int(np.prod(self.shape)) if self.shape else 1

    def ptr(self) -> int:
        return self.data.data_ptr()


@dataclass
class AttnOpts:
    """rust/src/backend.rs:59-69: query / key positions, score scale, sliding
    window (0 = none) and attention soft-cap (0 = none)."""

    q_pos: Sequence[int]
    k_pos: Sequence[int]
    scale: float = 1.0
    sliding_window: int = 0
    attn_softcap: float = 0.0


@dataclass
class KvAppend:
    """rust/src/backend.rs:71-77: the grown tensor and the one it superseded."""

    tensor: GqTensor
    dead: Optional[GqTensor] = None


@dataclass
class KvPages:
    """One layer's pages of a paged key-value cache (gq_kv_pages, include/gq.h): ``k`` and
    ``v`` are cuda tensors [n_pages, heads, page_size, head_dim] of one type (float32,
    float16, bfloat16 or float8_e4m3fn), or [n_pages, heads, page_size, head_dim / 16 * 9]
    uint8 (rows of 4-bit values and their scales, GQ_KV_E2M1), kept alive here. Made by
    ``CudaBackend.kv_pages``."""

    k: object
    v: object
    struct: object = field(repr=False, default=None)
    ref: int = 0       # address of struct
    row: int = 0       # values of a token: heads * head_dim
    head_dim: int = 0


class Chain:
    """A created decode chain (gq_chain): run() enqueues it on the backend's
    stream (recordable into a graph), reset() clears its counters after a
    timed-out run, close() frees it."""

    def __init__(self, backend: "CudaBackend", handle: c_void_p):
        self.backend = backend
        self.handle = handle

    def run(self) -> None:
        self.backend._check(self.backend.lib.gq_chain_run(self.handle), "chain_run")

    def reset(self) -> None:
        self.backend._check(self.backend.lib.gq_chain_reset(self.handle), "chain_reset")

    def close(self) -> None:
        if self.handle is not None and self.handle.value:
            self.backend.lib.gq_chain_destroy(self.handle)
        self.handle = None


class CudaBackend:
    """The Backend-trait surface of the quantized hot path, on one CUDA device."""

    def __init__(self, device: int = 0, own_stream: bool = False):
        """own_stream=False runs on torch's current stream of the device;
        True keeps the context's own non-blocking stream (needed to record graphs)."""
        import torch  # device memory + streams (plumbing only)

        self._torch = torch
        self.lib = _abi.load()
        self.device = int(device)
        self.torch_device = torch.device("cuda", self.device)
        ctx = c_void_p()
        rc = self.lib.gq_ctx_create(self.device, ctypes.byref(ctx))
        if rc != _abi.GQ_OK:
            raise GqError(rc, f"gq_ctx_create(device={device}) failed: {self.lib.gq_status_string(rc).decode()}")
        self.ctx = ctx
        self._frame: list = []
        self._qweights: list = []
        self.own_stream = own_stream
        if not own_stream:
            self._bind_stream()

    # ---- plumbing ---------------------------------------------------------
    def _bind_stream(self) -> None:
        s = self._torch.cuda.current_stream(self.torch_device).cuda_stream
        # torch's default stream is the legacy NULL stream (handle 0); pass it as
        # cudaStreamLegacy (0x1), since NULL means "the context's own stream" here
        if not s:
            s = 1
        _abi.check(self.lib.gq_ctx_set_stream(self.ctx, c_void_p(s)), self.ctx, "set_stream")

    def _check(self, rc: int, what: str) -> None:
        _abi.check(rc, self.ctx, what)

    def _alloc(self, shape) -> GqTensor:
        t = self._torch.empty(tuple(shape), dtype=self._torch.float32, device=self.torch_device)
        g = GqTensor(shape=tuple(shape), data=t)
        self._frame.append(g)
        return g

    def _fresh(self, make, *shape, dtype):
        """make (torch.zeros or torch.empty) a new tensor that a call is about to write. Where
        the backend's stream is not torch's current one it is made on the backend's: filled
        ahead of the call, out of memory that only that stream's work is given once the caller
        lets go of it. What torch's stream still does with such memory is waited for (not
        while the stream is recorded: keep what a recorded call returns as long as its graph)."""
        torch = self._torch
        if self.torch_device.type == "cuda":
            callers = torch.cuda.current_stream(self.torch_device)
            if (callers.cuda_stream or 1) != self.stream_ptr():  # (1: the legacy default stream, as the backend has it)
                mine = self.torch_stream()
                with torch.cuda.stream(mine):
                    if not torch.cuda.is_current_stream_capturing():
                        mine.wait_stream(callers)
                    return make(*shape, dtype=dtype, device=self.torch_device)
        return make(*shape, dtype=dtype, device=self.torch_device)

    def close(self) -> None:
        if getattr(self, "ctx", None):
            for q in self._qweights:
                self.lib.gq_qweight_free(q)
            self._qweights.clear()
            self.lib.gq_ctx_destroy(self.ctx)
            self.ctx = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def name(self) -> str:
        return "cuda-b200"

    def num_sms(self) -> int:
        return self.lib.gq_ctx_num_sms(self.ctx)

    def stream_ptr(self) -> int:
        return int(self.lib.gq_ctx_get_stream(self.ctx) or 0)

    def torch_stream(self):
        """The backend's stream as one of torch's."""
        ptr, cuda = self.stream_ptr(), self._torch.cuda
        # (torch has no external stream of the legacy default stream's handle)
        return cuda.default_stream(self.torch_device) if ptr == 1 else cuda.ExternalStream(ptr, device=self.torch_device)

    # ---- record / replay (include/gq.h gq_graph_*) ------------------------------
    def record(self, fn):
        """Record the ops `fn()` issues into a replayable graph (own_stream only)."""
        self._check(self.lib.gq_graph_begin(self.ctx), "graph_begin")
        try:
            fn()
        except BaseException:
            tmp = c_void_p()
            self.lib.gq_graph_end(self.ctx, ctypes.byref(tmp))
            if tmp.value:
                self.lib.gq_graph_destroy(tmp)
            raise
        out = c_void_p()
        self._check(self.lib.gq_graph_end(self.ctx, ctypes.byref(out)), "graph_end")
        return out

    def replay(self, graph) -> None:
        self._check(self.lib.gq_graph_launch(self.ctx, graph), "graph_launch")

    def destroy_graph(self, graph) -> None:
        self.lib.gq_graph_destroy(graph)

    # ---- decode chains (include/gq.h gq_chain_*) ------------------------------------
    def chain(self, ops) -> "Chain":
        """A decode chain over `ops`: tuples (mode, w, w2, x, y, b, b_offset, cap)
        with w/w2 quantized GqTensors (w2 None unless mode 1), x/y/b device
        pointers (int) or f32 GqTensors (b None unless mode 2). One activation row
        per op; `Chain.run()` issues them all as one launch."""
        arr = (_abi.ChainOp * len(ops))()
        for i, (mode, w, w2, x, y, b, b_off, cap) in enumerate(ops):
            ptr = lambda t: None if t is None else (t if isinstance(t, int) else t.ptr())
            arr[i] = _abi.ChainOp(int(mode), c_void_p(w.qw), c_void_p(w2.qw if w2 is not None else None),
                                  c_void_p(ptr(x)), c_void_p(ptr(y)), c_void_p(ptr(b)), int(b_off), float(cap))
        out = c_void_p()
        self._check(self.lib.gq_chain_create(self.ctx, arr, len(ops), ctypes.byref(out)), "chain_create")
        return Chain(self, out)

    # ---- construction (rust/src/backend.rs:94-98) ----------------------------
    def tensor(self, data, shape: Sequence[int]) -> GqTensor:
        arr = np.ascontiguousarray(np.asarray(data, dtype=np.float32).reshape(tuple(shape)))
        t = self._torch.from_numpy(arr).to(self.torch_device)
        return GqTensor(shape=tuple(shape), data=t)

    def from_torch(self, t) -> GqTensor:
        """Wrap an existing cuda float32 contiguous tensor (no copy)."""
        assert t.is_cuda and t.dtype == self._torch.float32 and t.is_contiguous()
        return GqTensor(shape=tuple(t.shape), data=t)

    def quant_tensor(self, q: QuantWeight) -> GqTensor:
        qb = np.ascontiguousarray(np.asarray(q.qbytes, dtype=np.uint8))
        sc = np.ascontiguousarray(np.asarray(q.scales, dtype=np.float32))
        out = c_void_p()
        n, k = q.shape
        rc = self.lib.gq_qweight_upload(
            self.ctx, qb.ctypes.data_as(ctypes.POINTER(c_uint8)), qb.size,
            sc.ctypes.data_as(ctypes.POINTER(c_float)), sc.size, n, k, q.bits, int(bool(q.signed_i8)),
            q.group_size, ctypes.byref(out))
        self._check(rc, "quant_tensor")
        self._qweights.append(out.value)
        return GqTensor(shape=(n, k), qw=out.value, quant=q)

    def quant_tensor_from_device(self, qbytes_dev, scales, shape, bits: int, signed_i8: bool,
                                 group_size: int) -> GqTensor:
        """WgpuBackend::quant_tensor_from_gpu (rust/src/backend_wgpu.rs:447-456):
        the packed payload is a cuda uint8 tensor already on this device."""
        sc = np.ascontiguousarray(np.asarray(scales, dtype=np.float32))
        out = c_void_p()
        n, k = shape
        rc = self.lib.gq_qweight_upload_device(
            self.ctx, c_void_p(qbytes_dev.data_ptr()), qbytes_dev.numel(), sc.ctypes.data_as(ctypes.POINTER(c_float)),
            sc.size, n, k, bits, int(bool(signed_i8)), group_size, ctypes.byref(out))
        self._check(rc, "quant_tensor_from_device")
        self._qweights.append(out.value)
        return GqTensor(shape=(n, k), qw=out.value, quant=None)

    def free_quant(self, t: GqTensor) -> None:
        if t.qw in self._qweights:
            self._qweights.remove(t.qw)
            self.lib.gq_qweight_free(t.qw)
            t.qw = None

    def zeros(self, shape: Sequence[int]) -> GqTensor:
        t = self._torch.zeros(tuple(shape), dtype=self._torch.float32, device=self.torch_device)
        return GqTensor(shape=tuple(shape), data=t)

    def reshape(self, x: GqTensor, shape: Sequence[int]) -> GqTensor:
        if x.qw is not None:
            return GqTensor(shape=tuple(shape), qw=x.qw, quant=x.quant)
        return GqTensor(shape=tuple(shape), data=x.data.view(tuple(shape)))

    # ---- ops ------------------------------------------------------------------
    def _xm(self, x: GqTensor):
        k = x.shape[-1]
        m = x.size() // k if k else 0
        return m, k

    def linear(self, x: GqTensor, w: GqTensor) -> GqTensor:
        """y = x · Wᵀ; x [M, K], W [N, K] quantized (rust/src/backend.rs:105-106)."""
        self._require_quant(w, "linear")
        m, k = self._xm(x)
        y = self._alloc((m, w.shape[0]))
        self._check(self.lib.gq_linear(self.ctx, c_void_p(x.ptr()), m, k, c_void_p(w.qw), c_void_p(y.ptr())),
                    "linear")
        return y

    def linear_geglu(self, x: GqTensor, w_gate: GqTensor, w_up: GqTensor) -> GqTensor:
        """gelu(x · Wgᵀ) * (x · Wuᵀ) (rust/src/backend.rs:155-160)."""
        self._require_quant(w_gate, "linear_geglu")
        self._require_quant(w_up, "linear_geglu")
        m, k = self._xm(x)
        y = self._alloc((m, w_gate.shape[0]))
        self._check(self.lib.gq_linear_geglu(self.ctx, c_void_p(x.ptr()), m, k, c_void_p(w_gate.qw),
                                             c_void_p(w_up.qw), c_void_p(y.ptr())), "linear_geglu")
        return y

    def linear_gelu_mul_cols(self, x: GqTensor, w: GqTensor, b: GqTensor, offset: int) -> GqTensor:
        """gelu(x · Wᵀ) * b[:, offset:offset+N], b [M, stride] (rust/src/backend.rs:161-167)."""
        self._require_quant(w, "linear_gelu_mul_cols")
        m, k = self._xm(x)
        if len(b.shape) != 2 or b.shape[0] != m:
            raise GqError(_abi.GQ_ERR_INVALID_ARGUMENT, "linear_gelu_mul_cols: b must be [M, stride]")
        y = self._alloc((m, w.shape[0]))
        self._check(self.lib.gq_linear_gelu_mul_cols(self.ctx, c_void_p(x.ptr()), m, k, c_void_p(w.qw),
                                                     c_void_p(b.ptr()), b.shape[1], offset, c_void_p(y.ptr())),
                    "linear_gelu_mul_cols")
        return y

    def linear_softcap(self, x: GqTensor, w: GqTensor, cap: float, out: Optional[GqTensor] = None,
                       col0: int = 0) -> GqTensor:
        """softcap(linear(x, w), cap) in one pass — the lm_head of rust/src/model.rs:192
        followed by Backend::softcap. ``out``/``col0`` write a vocab shard into its
        column slice of a wider logits tensor."""
        self._require_quant(w, "linear_softcap")
        m, k = self._xm(x)
        y = out if out is not None else self._alloc((m, w.shape[0]))
        ldy = y.shape[-1]
        self._check(self.lib.gq_linear_softcap(self.ctx, c_void_p(x.ptr()), m, k, c_void_p(w.qw), float(cap),
                                               c_void_p(y.ptr()), ldy, col0), "linear_softcap")
        return y

    def embed_rows(self, table: GqTensor, ids: Sequence[int], scale: float) -> GqTensor:
        """out[i, :] = deq(table)[ids[i], :] * scale (rust/src/backend.rs:101-102)."""
        self._require_quant(table, "embed_rows")
        if isinstance(ids, self._torch.Tensor) and ids.is_cuda:
            dids = ids.to(self._torch.int32).contiguous()
        else:
            arr = np.ascontiguousarray(np.asarray(ids, dtype=np.uint32))
            dids = self._torch.from_numpy(arr.view(np.int32)).to(self.torch_device)
        t = int(dids.numel())
        out = self._alloc((t, table.shape[1]))
        self._check(self.lib.gq_embed_rows(self.ctx, c_void_p(table.qw), c_void_p(dids.data_ptr()), t,
                                           float(scale), c_void_p(out.ptr())), "embed_rows")
        self._frame.append(GqTensor(shape=(t,), data=dids))  # keep ids alive until the frame ends
        return out

    def softcap(self, a: GqTensor, cap: float) -> GqTensor:
        y = self._alloc(a.shape)
        self._check(self.lib.gq_softcap(self.ctx, c_void_p(a.ptr()), a.size(), float(cap), c_void_p(y.ptr())),
                    "softcap")
        return y

    def geglu(self, gate: GqTensor, up: GqTensor) -> GqTensor:
        y = self._alloc(gate.shape)
        self._check(self.lib.gq_geglu(self.ctx, c_void_p(gate.ptr()), c_void_p(up.ptr()), gate.size(),
                                      c_void_p(y.ptr())), "geglu")
        return y

    # ---- support ops of a decode step (rust/src/backend.rs:103-154) ------------
    def _u32_dev(self, vals):
        if isinstance(vals, self._torch.Tensor) and vals.is_cuda:
            t = vals.to(self._torch.int32).contiguous()
        else:
            arr = np.ascontiguousarray(np.asarray(vals, dtype=np.uint32))
            t = self._torch.from_numpy(arr.view(np.int32)).to(self.torch_device)
        self._frame.append(GqTensor(shape=(t.numel(),), data=t))  # alive until the frame ends
        return t

    def tensor_bf16(self, data, shape: Sequence[int]) -> GqTensor:
        """A plain weight stored as bf16 (round to nearest even; exact for values that
        are bf16 on disk, like the reference's BF16 checkpoint tensors)."""
        arr = np.ascontiguousarray(np.asarray(data, dtype=np.float32).reshape(tuple(shape)))
        u = arr.view(np.uint32)
        rounded = ((u + np.uint32(0x7FFF) + ((u >> np.uint32(16)) & np.uint32(1))) >> np.uint32(16)).astype(np.uint16)
        t = self._torch.from_numpy(rounded.view(np.int16)).to(self.torch_device)
        return GqTensor(shape=tuple(shape), data=t, bf16=True)

    def rms_norm(self, x: GqTensor, w: Optional[GqTensor], eps: float) -> GqTensor:
        """y = x / sqrt(mean(x²) + eps) * w per row (rust/src/backend.rs:103-104)."""
        d = x.shape[-1]
        y = self._alloc(x.shape)
        self._check(self.lib.gq_rms_norm(self.ctx, c_void_p(x.ptr()), x.size() // d, d,
                                         c_void_p(w.ptr()) if w is not None else None, float(eps),
                                         c_void_p(y.ptr()), d), "rms_norm")
        return y

    def add_rms_norm(self, residual: GqTensor, x: GqTensor, w: GqTensor, eps: float,
                     scale_by: Optional[GqTensor] = None) -> GqTensor:
        """(residual + rms_norm(x, w)) * scale_by[0] (rust/src/backend.rs:137-144)."""
        d = x.shape[-1]
        y = self._alloc(x.shape)
        self._check(self.lib.gq_add_rms_norm(self.ctx, c_void_p(residual.ptr()), c_void_p(x.ptr()), x.size() // d,
                                             d, c_void_p(w.ptr()), float(eps),
                                             c_void_p(scale_by.ptr()) if scale_by is not None else None,
                                             c_void_p(y.ptr())), "add_rms_norm")
        return y

    def head_norm_rope(self, x: GqTensor, w: GqTensor, eps: float, positions, theta: float, head_dim: int,
                       heads: int, rotary_dim: int) -> GqTensor:
        """Per-head weighted RMSNorm then partial RoPE (rust/src/backend.rs:148-154)."""
        pos = self._u32_dev(positions)
        t = x.size() // (heads * head_dim)
        y = self._alloc(x.shape)
        self._check(self.lib.gq_head_norm_rope(self.ctx, c_void_p(x.ptr()), t, heads, head_dim, c_void_p(w.ptr()),
                                               float(eps), c_void_p(pos.data_ptr()), float(theta), rotary_dim,
                                               c_void_p(y.ptr()), 0), "head_norm_rope")
        return y

    def rope(self, x: GqTensor, positions, theta: float, head_dim: int, heads: int, rotary_dim: int) -> GqTensor:
        """Half-split partial RoPE on [T, heads, head_dim] (rust/src/backend.rs:118-119)."""
        pos = self._u32_dev(positions)
        t = x.size() // (heads * head_dim)
        y = self._alloc(x.shape)
        self._check(self.lib.gq_rope(self.ctx, c_void_p(x.ptr()), t, heads, head_dim, c_void_p(pos.data_ptr()),
                                     float(theta), rotary_dim, c_void_p(y.ptr()), 0), "rope")
        return y

    def attention(self, q: GqTensor, k: GqTensor, v: GqTensor, opts: AttnOpts) -> GqTensor:
        """q [T, Hq, Dh], k/v [S, Hkv, Dh] -> [T, Hq*Dh] (rust/src/backend.rs:120-121)."""
        t, hq, dh = q.shape
        s, hkv = k.shape[0], k.shape[1]
        if v.shape[-1] != dh or k.shape[-1] != dh:
            raise GqError(_abi.GQ_ERR_UNSUPPORTED, "attention: value head_dim must equal key head_dim")
        qp, kp = self._u32_dev(opts.q_pos), self._u32_dev(opts.k_pos)
        kpos = np.asarray(opts.k_pos, dtype=np.int64)
        flags = _abi.GQ_ATTN_KPOS_ASCENDING if (kpos.size < 2 or bool(np.all(np.diff(kpos) > 0))) else 0
        y = self._alloc((t, hq * dh))
        self._check(self.lib.gq_attention(self.ctx, c_void_p(q.ptr()), 1, t, hq, dh, c_void_p(k.ptr()),
                                          c_void_p(v.ptr()), s, hkv, 0, c_void_p(qp.data_ptr()),
                                          c_void_p(kp.data_ptr()), 0, float(opts.scale), int(opts.sliding_window),
                                          float(opts.attn_softcap), flags, c_void_p(y.ptr())), "attention")
        return y

    def linear_plain(self, x: GqTensor, w: GqTensor) -> GqTensor:
        """linear with a plain (bf16-stored) weight [N, K] (rust/src/backend_cpu.rs:174-222)."""
        if not w.bf16:
            raise GqError(_abi.GQ_ERR_INVALID_ARGUMENT, "linear_plain: weight must come from tensor_bf16")
        m, k = self._xm(x)
        n = w.shape[0]
        y = self._alloc((m, n))
        self._check(self.lib.gq_linear_bf16(self.ctx, c_void_p(x.ptr()), m, k, c_void_p(w.ptr()), n,
                                            c_void_p(y.ptr())), "linear_bf16")
        return y

    def _ew(self, fn, *args, shape, what):
        y = self._alloc(shape)
        self._check(fn(self.ctx, *args, c_void_p(y.ptr())), what)
        return y

    def add(self, a: GqTensor, b: GqTensor) -> GqTensor:
        return self._ew(self.lib.gq_add, c_void_p(a.ptr()), c_void_p(b.ptr()), a.size(), shape=a.shape, what="add")

    def mul(self, a: GqTensor, b: GqTensor) -> GqTensor:
        return self._ew(self.lib.gq_mul, c_void_p(a.ptr()), c_void_p(b.ptr()), a.size(), shape=a.shape, what="mul")

    def scale(self, a: GqTensor, s: float) -> GqTensor:
        return self._ew(self.lib.gq_scale, c_void_p(a.ptr()), a.size(), float(s), shape=a.shape, what="scale")

    def scale_by_tensor(self, a: GqTensor, s: GqTensor) -> GqTensor:
        return self._ew(self.lib.gq_scale_by_tensor, c_void_p(a.ptr()), a.size(), c_void_p(s.ptr()), shape=a.shape,
                        what="scale_by_tensor")

    def _copy_rows(self, src: GqTensor, rows: int, cols: int, src_stride: int, src_off: int, dst: GqTensor,
                   dst_stride: int, dst_off: int) -> None:
        self._check(self.lib.gq_copy_rows(self.ctx, c_void_p(src.ptr() + 4 * src_off), rows, cols, src_stride,
                                          c_void_p(dst.ptr() + 4 * dst_off), dst_stride), "copy_rows")

    def slice_rows(self, x: GqTensor, start: int, count: int) -> GqTensor:
        """Rows [start, start+count) of [rows, dim] (rust/src/backend.rs:122-123)."""
        dim = x.shape[1]
        y = self._alloc((count, dim))
        self._copy_rows(x, count, dim, dim, start * dim, y, dim, 0)
        return y

    def slice_cols(self, x: GqTensor, offset: int, width: int) -> GqTensor:
        """[:, offset:offset+width] of [rows, stride] (rust/src/backend.rs:124-125)."""
        rows, stride = x.shape
        y = self._alloc((rows, width))
        self._copy_rows(x, rows, width, stride, offset, y, width, 0)
        return y

    def concat_rows(self, a: Optional[GqTensor], b: GqTensor) -> GqTensor:
        """Concatenate along dim 0 (rust/src/backend.rs:126-127)."""
        if a is None:
            y = self._alloc(b.shape)
            self._copy_rows(b, 1, b.size(), b.size(), 0, y, b.size(), 0)
            return y
        shape = (a.shape[0] + b.shape[0],) + tuple(a.shape[1:])
        y = self._alloc(shape)
        self._copy_rows(a, 1, a.size(), a.size(), 0, y, a.size(), 0)
        self._copy_rows(b, 1, b.size(), b.size(), 0, y, b.size(), a.size())
        return y

    def kv_append(self, existing: Optional[GqTensor], add: GqTensor) -> KvAppend:
        """Append rows (rust/src/backend.rs:128-130): a new tensor holding old ++ new;
        the old one is reported dead, as on the CPU backend."""
        return KvAppend(tensor=self.concat_rows(existing, add), dead=existing)

    # ---- paged cache and logits of many requests (include/gq.h) -------------------
    # Device tensors here are torch tensors (rows of f32, i.e. k, v, q, logits and out, may be
    # GqTensors); the calls check types, devices and shapes, and the library the rest.
    def kv_pages(self, k, v, k_scale: float = 1.0, v_scale: float = 1.0) -> KvPages:
        """Describe one layer's pages: k, v [n_pages, heads, page_size, head_dim] of the same
        shape, strides and type; a page's values are contiguous, pages may lie apart. uint8:
        4-bit values, rows of head_dim / 16 * 9 bytes (GQ_KV_E2M1)."""
        torch = self._torch
        types = {torch.float32: _abi.GQ_KV_F32, torch.float16: _abi.GQ_KV_F16, torch.bfloat16: _abi.GQ_KV_BF16,
                 torch.float8_e4m3fn: _abi.GQ_KV_E4M3, torch.uint8: _abi.GQ_KV_E2M1}
        if k.dtype not in types or v.dtype != k.dtype:
            raise GqError(_abi.GQ_ERR_UNSUPPORTED, f"kv_pages: types {k.dtype} and {v.dtype}")
        if k.dim() != 4 or k.shape != v.shape or k.device != self.torch_device or v.device != self.torch_device:
            raise GqError(_abi.GQ_ERR_INVALID_ARGUMENT,
                          "kv_pages: k and v must be [n_pages, heads, page_size, head_dim] on the backend's device")
        n, h, ps, d = k.shape
        apart = k.stride(0) if n > 1 else h * ps * d
        for t in (k, v):
            if t.numel() and (not t[0].is_contiguous() or (n > 1 and t.stride(0) != apart)):
                raise GqError(_abi.GQ_ERR_INVALID_ARGUMENT, "kv_pages: a page's values must be contiguous, k and v strided alike")
        if apart < h * ps * d:  # (an expanded tensor's stride 0 would mean packed pages to the library)
            raise GqError(_abi.GQ_ERR_INVALID_ARGUMENT, "kv_pages: pages lie on one another")
        if k.dtype == torch.uint8:
            if d % 9 != 0:
                raise GqError(_abi.GQ_ERR_INVALID_ARGUMENT, "kv_pages: rows of 4-bit values are head_dim / 16 * 9 bytes")
            d = d // 9 * 16
        st = _abi.KvPagesStruct(k.data_ptr(), v.data_ptr(), n, ps, h, d, apart, types[k.dtype], float(k_scale), float(v_scale))
        return KvPages(k, v, st, ctypes.addressof(st), h * d, d)

    # (Single calls of these ops take the GPU 2-9 us, as long as the checks and the
    # conversions of 8-19 arguments take the host: the checks below ask for as little as
    # they can, and only a failed one says what was wrong.)
    def _dev(self, t, dtype, what: str, numel: int = 0) -> int:
        """Pointer of a contiguous device tensor of at least numel elements, checked."""
        if t.dtype is not dtype or t.get_device() != self.device or not t.is_contiguous() or t.numel() < numel:
            raise GqError(_abi.GQ_ERR_INVALID_ARGUMENT,
                          f"{what} must be a contiguous {dtype} tensor of at least {numel} elements on the backend's device")
        return t.data_ptr()

    def _rows(self, x, rows: int, width: int, what: str):
        """A f32 device tensor of `rows` rows as (pointer, row stride): rows may lie apart, a
        row's `width` values are contiguous."""
        t = x.data if isinstance(x, GqTensor) else x
        if t.dtype is not self._torch.float32 or t.get_device() != self.device or t.numel() != rows * width:
            raise GqError(_abi.GQ_ERR_INVALID_ARGUMENT,
                          f"{what} must be {rows} rows of {width} float32 values on the backend's device")
        if t.is_contiguous():
            return t.data_ptr(), width
        if t.dim() < 2 or t.shape[0] != rows or not t[0].is_contiguous() or t.stride(0) < width:
            raise GqError(_abi.GQ_ERR_INVALID_ARGUMENT, f"{what}: a row must be {width} contiguous values, rows apart")
        return t.data_ptr(), t.stride(0)

    def _table(self, block_table, batch: int, what: str):
        shape = block_table.shape
        if len(shape) != 2 or shape[0] < batch:
            raise GqError(_abi.GQ_ERR_INVALID_ARGUMENT, f"{what}: block_table must be [batch, pages]")
        return self._dev(block_table, self._torch.int32, "block_table"), shape[1]

    def paged_reserve(self, seq_lens, new_lens, page_size: int, block_table, free_pages, free_count, slots, positions,
                      owners, totals, free_left) -> None:
        """Take pages for each request's new tokens and number the tokens (gq_paged_reserve):
        int32 device tensors, slots int64; slots, positions and owners have one place per
        token of the (padded) step; totals may be seq_lens and free_left free_count."""
        d, i32, n, m = self._dev, self._torch.int32, seq_lens.numel(), slots.numel()
        tp, width = self._table(block_table, n, "paged_reserve")
        rc = self.lib.gq_paged_reserve(
            self.ctx, n, page_size, d(seq_lens, i32, "seq_lens"), d(new_lens, i32, "new_lens", n), tp, width,
            d(free_pages, i32, "free_pages"), free_pages.numel(), d(free_count, i32, "free_count", 1),
            d(free_left, i32, "free_left", 1), m, d(slots, self._torch.int64, "slots"), d(positions, i32, "positions", m),
            d(owners, i32, "owners", m), d(totals, i32, "totals", n))
        if rc:
            self._check(rc, "paged_reserve")

    def paged_release(self, seq_lens, keep_lens, page_size: int, block_table, free_pages, free_count, totals,
                      free_left) -> None:
        """Give back the pages past each request's keep_lens tokens (gq_paged_release)."""
        d, i32, n = self._dev, self._torch.int32, seq_lens.numel()
        tp, width = self._table(block_table, n, "paged_release")
        rc = self.lib.gq_paged_release(
            self.ctx, n, page_size, d(seq_lens, i32, "seq_lens"), d(keep_lens, i32, "keep_lens", n), tp, width,
            d(free_pages, i32, "free_pages"), free_pages.numel(), d(free_count, i32, "free_count", 1),
            d(free_left, i32, "free_left", 1), d(totals, i32, "totals", n))
        if rc:
            self._check(rc, "paged_release")

    def paged_append(self, pages: KvPages, k, v, slots) -> None:
        """Write rows k, v [T, heads, head_dim] f32 (token strides free) to slots [T] int64
        of the pages, rounded to their type (gq_paged_append)."""
        n = slots.numel()
        if pages.row != pages.head_dim:  # (several heads: rows by head would be in another order)
            for x in (k, v):
                shape = x.shape
                if len(shape) > 2 and shape[-1] * shape[-2] != pages.row:
                    raise GqError(_abi.GQ_ERR_INVALID_ARGUMENT, "paged_append: k and v must be [T, heads, head_dim]")
        kp, ks = self._rows(k, n, pages.row, "paged_append: k")
        vp, vs = self._rows(v, n, pages.row, "paged_append: v")
        rc = self.lib.gq_paged_append(self.ctx, pages.ref, kp, vp, n, ks, vs, self._dev(slots, self._torch.int64, "slots"))
        if rc:
            self._check(rc, "paged_append")

    def paged_read(self, pages: KvPages, slots, k_out=None, v_out=None):
        """The rows at slots [T] int64 of the pages as f32 k, v [T, heads, head_dim]
        (gq_paged_read): `k_out` and `v_out` (token strides free), whose rows of negative
        slots stay as they are, or new tensors, where such rows are 0."""
        n, heads = slots.numel(), pages.struct.heads
        new = lambda: self._fresh(self._torch.zeros, n, heads, pages.head_dim, dtype=self._torch.float32)  # noqa: E731
        k, v = k_out if k_out is not None else new(), v_out if v_out is not None else new()
        if pages.row != pages.head_dim:  # (as in paged_append)
            for x in (k, v):
                shape = x.shape
                if len(shape) > 2 and shape[-1] * shape[-2] != pages.row:
                    raise GqError(_abi.GQ_ERR_INVALID_ARGUMENT, "paged_read: k_out and v_out must be [T, heads, head_dim]")
        kp, ks = self._rows(k, n, pages.row, "paged_read: k_out")
        vp, vs = self._rows(v, n, pages.row, "paged_read: v_out")
        rc = self.lib.gq_paged_read(self.ctx, pages.ref, self._dev(slots, self._torch.int64, "slots"), n, kp, vp, ks, vs)
        if rc:
            self._check(rc, "paged_read")
        return k, v

    def paged_attention(self, pages: KvPages, q, block_table, seq_lens, scale: float = 1.0, sliding_window: int = 0,
                        attn_softcap: float = 0.0, out=None):
        """Attention of one new token per request over its pages (gq_paged_attention):
        q [batch, hq, head_dim] f32 (token stride free), block_table [batch, pages] and
        seq_lens [batch] int32 -> [batch, hq * head_dim] (`out`, or a new tensor)."""
        t = q.data if isinstance(q, GqTensor) else q
        batch, shape = seq_lens.numel(), t.shape
        if len(shape) != 3 or shape[0] != batch or shape[2] != pages.head_dim:
            raise GqError(_abi.GQ_ERR_INVALID_ARGUMENT, "paged_attention: q must be [batch, hq, head_dim]")
        hq = shape[1]
        width = hq * shape[2]
        qp, qs = self._rows(t, batch, width, "paged_attention: q")
        tp, entries = self._table(block_table, batch, "paged_attention")
        y = out if out is not None else self._alloc((batch, width))
        yt = y.data if isinstance(y, GqTensor) else y
        rc = self.lib.gq_paged_attention(
            self.ctx, pages.ref, qp, batch, hq, qs, tp, entries, self._dev(seq_lens, self._torch.int32, "seq_lens"), scale,
            sliding_window, attn_softcap, self._dev(yt, self._torch.float32, "out", batch * width))
        if rc:
            self._check(rc, "paged_attention")
        return y

    def process_logits(self, logits, tokens=None, prompt_lens=None, lens=None, penalties=None, bias_ids=None,
                       bias_values=None, bias_offsets=None, masks=None, mask_rows=None, out=None):
        """Repetition, presence and frequency penalties, biases and grammar masks of each row
        of logits [m, vocab] (gq_process_logits); `out` (may be the logits) or a new
        tensor. tokens [m, n] int32 with prompt_lens, lens [m] int32 and penalties [m, 3]
        f32; biases as bias_ids int32, bias_values f32 and bias_offsets [m + 1] int32;
        masks [k, ceil(vocab / 32)] int32 words with mask_rows [m] int32."""
        torch, d = self._torch, self._dev
        i32, f32 = torch.int32, torch.float32
        lt = logits.data if isinstance(logits, GqTensor) else logits
        shape = lt.shape
        if len(shape) != 2:
            raise GqError(_abi.GQ_ERR_INVALID_ARGUMENT, "process_logits: logits must be [m, vocab]")
        m, vocab = shape
        lp, ld = self._rows(lt, m, vocab, "process_logits: logits")
        y = out if out is not None else self._alloc((m, vocab))
        yt = y.data if isinstance(y, GqTensor) else y
        if yt.shape != shape:
            raise GqError(_abi.GQ_ERR_INVALID_ARGUMENT, "process_logits: out must have the logits' shape")
        yp, ldy = self._rows(yt, m, vocab, "process_logits: out")
        tok = pl = ln = pen = bi = bv = bo = mk = mr = None
        n_tok = n_masks = words = n_bias = 0
        if tokens is not None and tokens.numel():
            ts = tokens.shape
            if len(ts) != 2 or ts[0] != m or prompt_lens is None or lens is None or penalties is None:
                raise GqError(_abi.GQ_ERR_INVALID_ARGUMENT,
                              "process_logits: tokens must be [m, n], with prompt_lens, lens and penalties")
            tok, n_tok = d(tokens, i32, "tokens"), ts[1]
            pl, ln = d(prompt_lens, i32, "prompt_lens", m), d(lens, i32, "lens", m)
            pen = d(penalties, f32, "penalties", 3 * m)
        if bias_offsets is not None and bias_ids is not None and bias_values is not None:
            if n_bias := bias_ids.numel():
                bi, bv = d(bias_ids, i32, "bias_ids"), d(bias_values, f32, "bias_values", n_bias)
                bo = d(bias_offsets, i32, "bias_offsets", m + 1)
        elif bias_offsets is not None or bias_ids is not None or bias_values is not None:
            raise GqError(_abi.GQ_ERR_INVALID_ARGUMENT, "process_logits: biases are bias_ids, bias_values and bias_offsets")
        if masks is not None and masks.numel():
            if masks.dim() != 2:
                raise GqError(_abi.GQ_ERR_INVALID_ARGUMENT, "process_logits: masks must be [k, words]")
            mk, (n_masks, words) = d(masks, i32, "masks"), masks.shape
            mr = d(mask_rows, i32, "mask_rows", m) if mask_rows is not None else None
        rc = self.lib.gq_process_logits_bounded(self.ctx, lp, m, vocab, ld, tok, n_tok, pl, ln, pen, bi, bv, bo, n_bias, mk,
                                                n_masks, words, mr, yp, ldy)
        if rc:
            self._check(rc, "process_logits")
        return y

    def sample_requests(self, logits, temperature=None, top_k=None, top_p=None, min_p=None, uniforms=None, rng_state=None,
                        tokens=None, probs=None):
        """A token for each row of logits [m, vocab], drawn with the row's own options
        (gq_sample_requests): temperature, top_p and min_p [m] f32, top_k [m] int32 (None:
        off), and uniforms [m] f64 in [0, 1) or rng_state [m] int64 (splitmix64 states,
        advanced). -> tokens [m] int32 (`tokens`, or a new tensor); `probs` [m] f32, when
        given, receives the probabilities that they were drawn with."""
        torch, d = self._torch, self._dev
        f32 = torch.float32
        lt = logits.data if isinstance(logits, GqTensor) else logits
        shape = lt.shape
        if len(shape) != 2:
            raise GqError(_abi.GQ_ERR_INVALID_ARGUMENT, "sample_requests: logits must be [m, vocab]")
        m, vocab = shape
        lp, ld = self._rows(lt, m, vocab, "sample_requests: logits")
        if tokens is None:
            tokens = self._fresh(torch.empty, m, dtype=torch.int32)
        rc = self.lib.gq_sample_requests(
            self.ctx, lp, m, vocab, ld, d(temperature, f32, "temperature", m) if temperature is not None else None,
            d(top_k, torch.int32, "top_k", m) if top_k is not None else None,
            d(top_p, f32, "top_p", m) if top_p is not None else None, d(min_p, f32, "min_p", m) if min_p is not None else None,
            d(uniforms, torch.float64, "uniforms", m) if uniforms is not None else None,
            d(rng_state, torch.int64, "rng_state", m) if rng_state is not None else None, d(tokens, torch.int32, "tokens", m),
            d(probs, f32, "probs", m) if probs is not None else None)
        if rc:
            self._check(rc, "sample_requests")
        return tokens

    # ---- sync / lifecycle (rust/src/backend.rs:169-179) ------------------------
    def readback(self, t: GqTensor) -> np.ndarray:
        """Blocking read of a tensor's f32 contents; raises on a device-reported error."""
        out = np.empty(t.size(), dtype=np.float32)
        self._check(self.lib.gq_readback(self.ctx, out.ctypes.data_as(c_void_p), c_void_p(t.ptr()), out.size),
                    "readback")
        return out

    def flush(self) -> None:
        self._check(self.lib.gq_sync(self.ctx), "flush")

    def begin_frame(self) -> None:
        self._frame = []

    def end_frame(self, keep: Sequence[GqTensor] = (), also_free: Sequence[GqTensor] = ()) -> None:
        keep_ids = {id(k.data) for k in keep if k.data is not None}
        self._frame = [t for t in self._frame if id(t.data) in keep_ids]
        for t in also_free:
            self.free_tensor(t)

    def free_tensor(self, t: GqTensor) -> None:
        if t.qw is not None:
            self.free_quant(t)
        t.data = None

    @staticmethod
    def _require_quant(w: GqTensor, op: str) -> None:
        if w.qw is None:
            raise GqError(_abi.GQ_ERR_INVALID_ARGUMENT, f"{op}: weight is not a quantized tensor")
