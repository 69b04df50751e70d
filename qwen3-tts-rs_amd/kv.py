"""Key/value cache with a page table in 16 or 8 bits, and attention of new tokens over it (qtts_kv_* of include/qtts.h).

For serving loops around transformer layers of the caller's own: tensors are torch tensors on the cache's GPU, work is enqueued on
torch's current stream of that GPU, nothing is waited for, and the calls can be captured into a graph.  The reference keeps a tensor
per layer inside the model (qwen_tts/src/nn/kv_cache.rs:38-42); `LoaderConfig.kv_cache` puts the talker's own cache in 8 bits.

    cache = KVCache(layers=28, pages=4096, kv_heads=8, head_dim=128, format="e4m3")
    step = cache.batch(new=[5, 1], ctx=[5, 213], page_table=table)    # once per step, for all layers
    cache.write(layer, step, k, v)                                    # (6, 8, 128) each, f32 or bf16
    out = cache.attend(layer, step, q)                                # (6, heads, 128) bf16
"""
from __future__ import annotations

import ctypes as C
from typing import Optional, Sequence

from . import _lib
from ._lib import KV_FORMATS, QTTS_BF16, QTTS_F32, QttsError, check


class KVBatch:
    """The sequences of a call (qtts_kv_batch): device int32 tensors q_start (n_seq + 1), ctx_len (n_seq) and page_table
    (n_seq, max_pages), and the host bounds on what they hold (a length beyond its bound is cut).  A captured call reads the tensors
    when it is replayed, so a serving loop may move the lengths on in place, up to max_ctx.  `KVCache.batch` makes one from host lists,
    with bounds that just hold them."""

    def __init__(self, q_start, ctx_len, page_table, n_tokens: int, max_new: int, max_ctx: int):
        import torch
        for name, t, dim in (("q_start", q_start, 1), ("ctx_len", ctx_len, 1), ("page_table", page_table, 2)):
            if not isinstance(t, torch.Tensor) or t.dtype != torch.int32 or t.dim() != dim or not t.is_contiguous():
                raise QttsError(-1, f"KVBatch: {name} must be a contiguous int32 tensor of {dim} dimension(s)")
        n = ctx_len.shape[0]
        if q_start.shape[0] != n + 1 or page_table.shape[0] != n:
            raise QttsError(-4, "KVBatch: q_start, ctx_len and page_table do not describe the same number of sequences")
        if not (q_start.device == ctx_len.device == page_table.device):
            raise QttsError(-1, "KVBatch: tensors on different devices")
        for name, x in (("n_tokens", n_tokens), ("max_new", max_new), ("max_ctx", max_ctx)):
            if not 0 <= int(x) < 1 << 31:
                raise QttsError(-1, f"KVBatch: {name} out of range")
        self.q_start, self.ctx_len, self.page_table = q_start, ctx_len, page_table
        self.n_seq, self.n_tokens, self.max_new, self.max_ctx = n, int(n_tokens), int(max_new), int(max_ctx)
        self.device = ctx_len.device
        self._c = _lib.KvBatch(n, self.n_tokens, self.max_new, self.max_ctx, page_table.shape[1], q_start.data_ptr(), ctx_len.data_ptr(),
                               page_table.data_ptr())
        self._ptr = C.addressof(self._c)
        self._ws = {}


class KVCache:
    """`layers` x `pages` pages of `page_tokens` tokens (qtts_kv_open); format "bf16", "e4m3" or "int8" (the 8-bit formats hold blocks
    of 32 elements with one power-of-two scale each)."""

    def __init__(self, pages: int, kv_heads: int, head_dim: int, format: str = "bf16", layers: int = 1, page_tokens: int = 64, device: int = 0):
        if format not in KV_FORMATS:
            raise QttsError(-1, f"KVCache: unknown format '{format}'. Available: {sorted(KV_FORMATS)}")
        import torch
        self._torch = torch
        self._f32, self._bf16 = torch.float32, torch.bfloat16
        self._forward_ad = torch.autograd.forward_ad
        # the stream's handle without a Stream object around it (2 us of a call's 10) where torch has that
        raw = getattr(torch._C, "_cuda_getCurrentRawStream", None)
        self._stream = (lambda: raw(int(device))) if raw else (lambda: torch.cuda.current_stream(self.device).cuda_stream)
        self.lib = _lib.load()
        self.layers, self.pages, self.page_tokens = int(layers), int(pages), int(page_tokens)
        self.kv_heads, self.head_dim, self.format = int(kv_heads), int(head_dim), format
        self.device = torch.device("cuda", int(device))
        self._ctx, self._kv = C.c_void_p(), C.c_void_p()
        current = torch.cuda.current_device() if torch.cuda.is_available() else None
        try:
            check(self.lib.qtts_init(int(device), C.byref(self._ctx)))
            cfg = _lib.KvConfig(self.layers, self.pages, self.page_tokens, self.kv_heads, self.head_dim, KV_FORMATS[format])
            check(self.lib.qtts_kv_open(self._ctx, C.byref(cfg), C.byref(self._kv)))
        except Exception:
            self.close()
            raise
        finally:
            if current is not None:
                torch.cuda.set_device(current)  # qtts_init made its GPU the current one

    def close(self):
        if getattr(self, "_kv", None):
            self.lib.qtts_kv_close(self._kv)
            self._kv = C.c_void_p()
        if getattr(self, "_ctx", None):
            self.lib.qtts_shutdown(self._ctx)
            self._ctx = C.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def bytes(self) -> int:
        """Device memory of the cache."""
        return int(self.lib.qtts_kv_bytes(self._kv))

    # ------------------------------------------------------------------ batches
    def batch(self, new: Sequence[int], ctx: Sequence[int], page_table) -> KVBatch:
        """Sequence b's last new[b] of ctx[b] tokens; page_table (n_seq, max_pages): an int32 tensor on the cache's GPU (copied if it
        is not contiguous), or host numbers.  The rows of the calls' tensors are the sequences' new tokens one after another."""
        import torch
        new, ctx = [int(x) for x in new], [int(x) for x in ctx]
        if len(new) != len(ctx) or any(n < 0 or n > c for n, c in zip(new, ctx)):
            raise QttsError(-1, "KVCache.batch: every sequence needs 0 <= new <= ctx")
        if not isinstance(page_table, torch.Tensor):
            page_table = torch.tensor(page_table, dtype=torch.int32).reshape(len(new), -1 if new else 0).to(self.device)
        start = [0]
        for n in new:
            start.append(start[-1] + n)
        dev = torch.tensor(start + ctx, dtype=torch.int32).to(self.device)
        b = KVBatch(dev[:len(start)], dev[len(start):], page_table.contiguous(), start[-1], max(new, default=0), max(ctx, default=0))
        if b.max_ctx > page_table.shape[1] * self.page_tokens:
            raise QttsError(-4, "KVCache.batch: a sequence is longer than its row of the page table")
        return b

    # ------------------------------------------------------------------ calls
    def _check(self, what, layer, batch, t, heads, dtypes):
        if not 0 <= layer < self.layers:
            raise QttsError(-1, f"{what}: no such layer")
        if not isinstance(batch, KVBatch):
            raise QttsError(-1, f"{what}: not a KVBatch")
        if not self._kv:
            raise QttsError(-5, f"{what}: the cache is closed")
        if batch.device != self.device or t.device != self.device:
            raise QttsError(-1, f"{what}: tensors must be on {self.device}")
        if t.dtype not in dtypes:
            raise QttsError(-1, f"{what}: dtype must be one of {[str(d) for d in dtypes]}")
        shape = tuple(t.shape)
        if len(shape) != 3 or shape[0] != batch.n_tokens or shape[2] != self.head_dim or (heads and shape[1] != heads):
            raise QttsError(-4, f"{what}: shape must be ({batch.n_tokens}, {heads or 'heads'}, {self.head_dim}), got {shape}")
        if t.stride(2) != 1 and t.numel():
            raise QttsError(-1, f"{what}: the elements of a head must be contiguous")
        if t.requires_grad and self._torch.is_grad_enabled():
            raise QttsError(-1, f"{what}: inference only, the tensor requires a gradient")
        if self._forward_ad._current_level >= 0 and self._forward_ad.unpack_dual(t).tangent is not None:
            raise QttsError(-1, f"{what}: inference only, the tensor has a tangent")

    def _move(self, call, layer, batch, k, v):
        r = _lib.KvRows(k.data_ptr(), v.data_ptr(), QTTS_F32 if k.dtype == self._f32 else QTTS_BF16, k.stride(0), k.stride(1), v.stride(0),
                        v.stride(1))
        check(call(self._kv, layer, batch._ptr, C.addressof(r), self._stream()))

    def write(self, layer: int, batch: KVBatch, k, v) -> None:
        """Holds the batch's tokens: k, v (n_tokens, kv_heads, head_dim), f32 or bf16."""
        self._check("KVCache.write", layer, batch, k, self.kv_heads, (self._bf16, self._f32))
        self._check("KVCache.write", layer, batch, v, self.kv_heads, (k.dtype,))
        self._move(self.lib.qtts_kv_write, layer, batch, k, v)

    def read(self, layer: int, batch: KVBatch, dtype=None, out=None):
        """The batch's tokens as they are held: (k, v), f32 or bf16 (the default); with new = ctx whole sequences.  out: a (k, v) pair
        to fill (rows behind the last sequence stay as they are)."""
        if out is None:
            if not isinstance(batch, KVBatch):
                raise QttsError(-1, "KVCache.read: not a KVBatch")
            k = self._torch.empty((batch.n_tokens, self.kv_heads, self.head_dim), dtype=dtype or self._bf16, device=self.device)
            out = k, self._torch.empty_like(k)
        k, v = out
        self._check("KVCache.read", layer, batch, k, self.kv_heads, (self._bf16, self._f32) if dtype is None else (dtype,))
        self._check("KVCache.read", layer, batch, v, self.kv_heads, (k.dtype,))
        if k.dtype != self._bf16 and k.dtype != self._f32:
            raise QttsError(-1, "KVCache.read: dtype must be float32 or bfloat16")
        self._move(self.lib.qtts_kv_read, layer, batch, k, v)
        return k, v

    def attend(self, layer: int, batch: KVBatch, q, scale: Optional[float] = None, window: int = 0, out=None):
        """softmax(scale q k^T) v of the batch's tokens over what the cache holds for their sequences: q (n_tokens, heads, head_dim)
        bf16, heads a multiple of kv_heads; scale defaults to head_dim ** -0.5.  A token sees the positions up to its own, with a
        window the last `window` of them.  out: a tensor to fill, which may be q itself.  The tokens' own keys and values have been written before."""
        self._check("KVCache.attend", layer, batch, q, 0, (self._bf16,))
        heads, window = q.shape[1], max(-1, min(int(window), 0x7fffffff))
        if out is None:
            out = self._torch.empty_like(q, memory_format=self._torch.contiguous_format)
        else:
            self._check("KVCache.attend: out", layer, batch, out, heads, (self._bf16,))
        shape = (self.kv_heads, self.head_dim, heads, window)
        nbytes = batch._ws.get(shape)
        if nbytes is None:
            n = C.c_int64(0)
            check(self.lib.qtts_kv_attend_workspace(self._kv, batch._ptr, heads, window, C.byref(n)))
            nbytes = batch._ws[shape] = n.value
        ws = self._torch.empty(nbytes, dtype=self._torch.uint8, device=self.device) if nbytes else None
        a = _lib.KvAttendArgs(q.data_ptr(), out.data_ptr(), q.stride(0), q.stride(1), out.stride(0), out.stride(1), heads,
                              self.head_dim ** -0.5 if scale is None else scale, window, ws.data_ptr() if nbytes else None, nbytes)
        check(self.lib.qtts_kv_attend(self._kv, layer, batch._ptr, C.addressof(a), self._stream()))
        return out
