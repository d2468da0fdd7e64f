"""An 8-bit paged KV cache for serving several sequences (vkq_kv8_*).

    cache = kv8.Cache(layers, num_pages, 64, kv_heads, 128, "int8")
    seqs = kv8.Sequences(cache, max_seqs, max_pages)
    seqs.extend(slots, new)                      # lengths and pages of the new tokens
    batch = seqs.batch(slots, tokens=T, cu_tokens=cu, max_tokens=n, max_len=bound)
    for layer in range(layers):
        q = cache.append(layer, batch, k, v, q=q, cos=cos, sin=sin, layout="half")
        o = cache.attend(layer, batch, q)
    seqs.fork(src, dst); seqs.free(slots); seqs.compact()

Every call runs on torch's current stream (or `stream`) and returns without a
host synchronisation; lengths, page numbers and free pages stay on the device.
With `stream` the inputs must be ready for it and live until it has used them,
and a result is ready for another stream once that has waited for this one.
"""
from __future__ import annotations

import math

import torch

from . import vkq
from .tensor import ROPE_LAYOUTS, check_int32, check_tables, dtype_code, empty_on, stream_of

FORMATS = {"int8": vkq.KV8_INT8, "e4m3": vkq.KV8_E4M3}
BLOCK = vkq.KV8_BLOCK


def _ptr(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


class Batch:
    """The sequences that a call works on: row slots[b] (default b) of `table`
    [rows, max_pages] and `lens` [rows]; the new tokens of sequence b are rows
    cu_tokens[b] .. cu_tokens[b + 1] - 1 of q, k, v (default: row b)."""

    def __init__(self, table: torch.Tensor, lens: torch.Tensor, cu_tokens: torch.Tensor | None = None,
                 slots: torch.Tensor | None = None, tokens: int | None = None, max_tokens: int = 1,
                 max_len: int | None = None):
        dev = table.device
        check_int32(table, (None, None), "table", dev)
        check_int32(lens, (table.shape[0],), "lens", dev)
        n = table.shape[0]
        if slots is not None:
            check_int32(slots, (None,), "slots", dev)
            n = slots.shape[0]
        if cu_tokens is not None:
            if slots is None:
                n = cu_tokens.shape[0] - 1
            check_int32(cu_tokens, (n + 1,), "cu_tokens", dev)
            if tokens is None:
                raise ValueError("tokens (rows of q, k and v) is needed with cu_tokens")
        self.tensors = (table, lens, slots, cu_tokens)  # kept alive: the struct holds their pointers
        self.device = dev
        self.tokens = n if tokens is None else tokens
        self.max_len = max_len
        self._page = 0  # the page size that struct.max_len is for
        self.struct = vkq.Kv8BatchStruct(_ptr(table), _ptr(lens), _ptr(slots), _ptr(cu_tokens), table.shape[0],
                                         table.shape[1], n, self.tokens, max_tokens, 0)

    def bounds(self, page: int) -> vkq.Kv8BatchStruct:
        """The struct for a cache of this page size: its length bound is that of the table unless one was given."""
        s = self.struct
        if page != self._page:
            s.max_len = s.max_pages * page if self.max_len is None else self.max_len
            self._page = page
        return s


class Cache:
    """The pool: codes [layers, num_pages, kv_heads, page_size, head_dim] of
    K and V (uint8 storage of int8 or e4m3) and a scale for every 16 tokens of
    a page and head [layers, num_pages, kv_heads, page_size / 16].  `buffers`
    (k, v, k_scale, v_scale) are used in place of new ones."""

    def __init__(self, layers: int, num_pages: int, page_size: int, kv_heads: int, head_dim: int, fmt: str = "int8",
                 device="cuda", buffers: tuple | None = None):
        if fmt not in FORMATS:
            raise ValueError(f"format {fmt!r}: one of {sorted(FORMATS)}")
        if page_size <= 0 or page_size % BLOCK:
            raise ValueError(f"page_size {page_size} is no multiple of {BLOCK}")
        codes = (layers, num_pages, kv_heads, page_size, head_dim)
        scales = (layers, num_pages, kv_heads, page_size // BLOCK)
        if buffers is None:
            buffers = (torch.zeros(codes, dtype=torch.uint8, device=device),
                       torch.zeros(codes, dtype=torch.uint8, device=device),
                       torch.ones(scales, device=device), torch.ones(scales, device=device))
        for t, shape, dt in zip(buffers, (codes, codes, scales, scales), (torch.uint8,) * 2 + (torch.float32,) * 2):
            if tuple(t.shape) != shape or t.dtype != dt or not t.is_contiguous() or not t.is_cuda or \
                    t.device != buffers[0].device:
                raise ValueError(f"a buffer is {tuple(t.shape)} {t.dtype} on {t.device}, {shape} {dt} contiguous needed")
        self.k, self.v, self.k_scale, self.v_scale = buffers
        self.layers, self.num_pages, self.page_size = layers, num_pages, page_size
        self.kv_heads, self.head_dim, self.fmt = kv_heads, head_dim, fmt
        self.device = self.k.device
        self.struct = vkq.Kv8CacheStruct(FORMATS[fmt], page_size, kv_heads, head_dim, layers, num_pages,
                                         *(t.data_ptr() for t in buffers))
        self._ws: dict[int, torch.Tensor] = {}
        self._captured: list[torch.Tensor] = []  # workspaces whose address a graph holds
        self._need: dict[tuple, int] = {}

    def _rows(self, t: torch.Tensor, batch: Batch, heads: int | None, name: str) -> tuple[int, int, int]:
        """Pointer, token stride and heads of activations [tokens, heads, head_dim]."""
        s = t.shape
        if len(s) != 3 or t.device != self.device or s[0] != batch.tokens or s[2] != self.head_dim or \
                (heads is not None and s[1] != heads):
            raise ValueError(f"{name} must be [{batch.tokens}, {heads or 'heads'}, {self.head_dim}] on {self.device}, "
                             f"got {tuple(s)} on {t.device}")
        st = t.stride()
        if s[0] and (st[2] != 1 or (s[1] > 1 and st[1] != s[2])):
            raise ValueError(f"the heads of a token must be contiguous in {name}")
        return t.data_ptr(), st[0] if s[0] > 1 else s[1] * s[2], s[1]

    def _bounds(self, batch: Batch) -> vkq.Kv8BatchStruct:
        if batch.device != self.device:
            raise ValueError(f"the batch is on {batch.device}, the cache on {self.device}")
        return batch.bounds(self.page_size)

    def append(self, layer: int, batch: Batch, k: torch.Tensor, v: torch.Tensor, q: torch.Tensor | None = None,
               cos: torch.Tensor | None = None, sin: torch.Tensor | None = None, layout: str = "interleaved",
               q_out: torch.Tensor | None = None, stream: torch.cuda.Stream | None = None) -> torch.Tensor | None:
        """Quantizes the new tokens' k and v [tokens, kv_heads, head_dim] into
        the pages of `layer`; with tables k is rotated first, and q [tokens,
        heads, head_dim] is returned rotated (q_out may be q)."""
        code = dtype_code(k)
        kp, ks, _ = self._rows(k, batch, self.kv_heads, "k")
        vp, vs, _ = self._rows(v, batch, self.kv_heads, "v")
        if v.dtype != k.dtype or (q is not None and q.dtype != k.dtype):
            raise ValueError("q, k and v must have one dtype")
        if (cos is None) != (sin is None) or (q is not None and cos is None):
            raise ValueError("both tables or neither, and both to rotate q")
        qp = qs = qop = qos = heads = seq = rot = 0
        if cos is not None:
            check_tables(cos, sin, self.device)
            seq, rot = cos.shape[0], 2 * cos.shape[1]
        if q is not None:
            qp, qs, heads = self._rows(q, batch, None, "q")
            if q_out is None:
                q_out = empty_on(q.shape, q.dtype, self.device, stream)
            elif q_out.dtype != q.dtype:
                raise ValueError("q_out must match q")
            qop, qos, _ = self._rows(q_out, batch, heads, "q_out")
        if batch.tokens == 0:
            return q_out
        vkq.kv8_append(self.struct, layer, self._bounds(batch), code, kp, ks, vp, vs, qp or None, qs,
                       qop or None, qos, heads, _ptr(cos), _ptr(sin), seq, rot, ROPE_LAYOUTS[layout],
                       device=self.device.index, stream=stream_of(self.device, stream))
        return q_out

    def read(self, layer: int, batch: Batch, seq: torch.Tensor, pos: torch.Tensor, dtype=torch.float32,
             stream: torch.cuda.Stream | None = None) -> tuple[torch.Tensor, torch.Tensor]:
        """K and V [n, kv_heads, head_dim] of sequence seq[i] of the batch at position pos[i]."""
        check_int32(seq, (None,), "seq", self.device)
        check_int32(pos, (seq.shape[0],), "pos", self.device)
        n = seq.shape[0]
        shape = (n, self.kv_heads, self.head_dim)
        k, v = (empty_on(shape, dtype, self.device, stream) for _ in range(2))
        if n:
            vkq.kv8_read(self.struct, layer, self._bounds(batch), seq.data_ptr(), pos.data_ptr(), n,
                         dtype_code(k), k.data_ptr(), v.data_ptr(), device=self.device.index,
                         stream=stream_of(self.device, stream))
        return k, v

    def workspace_bytes(self, batch: Batch, dtype: torch.dtype, heads: int, causal: bool = True, window: int = 0) -> int:
        """vkq_kv8_attention_workspace_bytes, memoised."""
        return self._needed(self._bounds(batch), dtype, heads, causal, window)

    def _needed(self, s: vkq.Kv8BatchStruct, dtype: torch.dtype, heads: int, causal: bool, window: int) -> int:
        key = (dtype, heads, causal, window, s.batch, s.max_tokens, s.max_len)
        need = self._need.get(key)
        if need is None:
            code = dtype_code(torch.empty(0, dtype=dtype))
            need = vkq.kv8_attention_workspace_bytes(self.struct, s, code, heads, causal, window,
                                                     device=self.device.index)
            self._need[key] = need
        return need

    def _capturing(self, stream: torch.cuda.Stream | None) -> bool:
        if stream is None and torch._C._cuda_getDevice() == self.device.index:  # asked for on every call: 0.4 us
            return torch._C._cuda_isCurrentStreamCapturing()
        with torch.cuda.stream(torch.cuda.current_stream(self.device) if stream is None else stream):
            return torch.cuda.is_current_stream_capturing()

    def _workspace(self, nbytes: int, stream: torch.cuda.Stream | None) -> torch.Tensor:
        """A zero-filled workspace of this cache and stream (calls on one stream
        may share it).  One that a capture has seen lives as long as the cache:
        its graph keeps the address."""
        key = stream_of(self.device, stream)
        ws = self._ws.get(key)
        capturing = self._capturing(stream)
        if ws is None or ws.numel() < nbytes:
            if capturing:
                raise RuntimeError("the workspace cannot grow in a stream capture: make the call once before on the "
                                   "stream that is captured (torch.cuda.graph(..., stream=s)), or give ws "
                                   "(zero-filled, workspace_bytes(...) long)")
            with torch.cuda.stream(stream):  # None: the current one
                ws = torch.zeros(max(nbytes, 1 << 20), dtype=torch.uint8, device=self.device)
            self._ws[key] = ws
        if capturing and not any(t is ws for t in self._captured):
            self._captured.append(ws)
        return ws

    def attend(self, layer: int, batch: Batch, q: torch.Tensor, scale: float | None = None, causal: bool = True,
               window: int = 0, out: torch.Tensor | None = None, ws: torch.Tensor | None = None,
               stream: torch.cuda.Stream | None = None) -> torch.Tensor:
        """Attention of the new tokens' q [tokens, heads, head_dim] over the
        cache (which holds them already); scale defaults to 1 / sqrt(head_dim).
        Without ws the cache's own workspace of this stream is used; a graph
        captured so keeps using it, and must not run at once with another
        graph of that stream or with calls on it."""
        code = dtype_code(q)
        qp, qs, heads = self._rows(q, batch, None, "q")
        if out is None:
            out = empty_on(q.shape, q.dtype, self.device, stream)
        elif out.dtype != q.dtype:
            raise ValueError("out must match q")
        op, os_, _ = self._rows(out, batch, heads, "out")
        if batch.tokens == 0:
            return out
        s = self._bounds(batch)
        if ws is None:
            ws = self._workspace(self._needed(s, q.dtype, heads, causal, window), stream)
            size = ws.numel()
        else:
            if ws.device != self.device or not ws.is_contiguous():
                raise ValueError(f"ws must be contiguous on {self.device}")
            size = ws.numel() * ws.element_size()
        vkq.kv8_attention(self.struct, layer, s, code, qp, qs, op, os_, heads,
                          1.0 / math.sqrt(self.head_dim) if scale is None else scale, ws.data_ptr(), size, causal, window,
                          device=self.device.index, stream=stream_of(self.device, stream))
        return out

    def copy_pages(self, src: torch.Tensor, dst: torch.Tensor, stream: torch.cuda.Stream | None = None) -> None:
        """The contents of pages src become those of pages dst, all layers."""
        check_int32(src, (None,), "src", self.device)
        check_int32(dst, (src.shape[0],), "dst", self.device)
        if src.shape[0]:
            vkq.kv8_copy_pages(self.struct, src.data_ptr(), dst.data_ptr(), src.shape[0], device=self.device.index,
                               stream=stream_of(self.device, stream))


class Sequences:
    """The bookkeeping of a cache's pages: table [max_seqs, max_pages] (-1: no
    page), lens [max_seqs] and refs [num_pages] (0: free).  Lists of rows are
    int32 device tensors of distinct rows."""

    def __init__(self, cache: Cache, max_seqs: int, max_pages: int, buffers: tuple | None = None):
        self.cache = cache
        if buffers is None:
            buffers = (torch.full((max_seqs, max_pages), -1, dtype=torch.int32, device=cache.device),
                       torch.zeros(max_seqs, dtype=torch.int32, device=cache.device),
                       torch.zeros(cache.num_pages, dtype=torch.int32, device=cache.device))
        self.table, self.lens, self.refs = buffers
        check_int32(self.table, (max_seqs, max_pages), "table", cache.device)
        check_int32(self.lens, (max_seqs,), "lens", cache.device)
        check_int32(self.refs, (cache.num_pages,), "refs", cache.device)
        self.struct = vkq.Kv8SeqsStruct(self.table.data_ptr(), self.lens.data_ptr(), self.refs.data_ptr(), max_seqs,
                                        max_pages)
        self._ws = torch.zeros(vkq.kv8_pages_workspace_bytes(cache.struct, self.struct), dtype=torch.uint8,
                               device=cache.device)

    def batch(self, slots: torch.Tensor | None = None, **kw) -> Batch:
        """The listed rows as a call's batch (see Batch)."""
        return Batch(self.table, self.lens, slots=slots, **kw)

    def _list(self, a: torch.Tensor, name: str, done: torch.Tensor | None) -> int:
        check_int32(a, (None,), name, self.cache.device)
        if done is not None:
            check_int32(done, (a.shape[0],), "done", self.cache.device)
        return a.shape[0]

    def extend(self, slots: torch.Tensor, add: torch.Tensor, done: torch.Tensor | None = None, stream=None) -> None:
        """Row slots[i] grows by add[i] tokens and the pages that it then needs;
        done[i]: whether it did (too few free pages: it stays as it was)."""
        n = self._list(slots, "slots", done)
        check_int32(add, (n,), "add", self.cache.device)
        if n:
            vkq.kv8_extend(self.cache.struct, self.struct, slots.data_ptr(), add.data_ptr(), n, _ptr(done),
                           self._ws.data_ptr(), self._ws.numel(), device=self.cache.device.index,
                           stream=stream_of(self.cache.device, stream))

    def fork(self, src: torch.Tensor, dst: torch.Tensor, done: torch.Tensor | None = None, stream=None) -> None:
        """The empty rows dst become copies of the rows src: whole pages shared, a part-filled last one copied."""
        n = self._list(dst, "dst", done)
        check_int32(src, (n,), "src", self.cache.device)
        if n:
            vkq.kv8_fork(self.cache.struct, self.struct, src.data_ptr(), dst.data_ptr(), n, _ptr(done),
                         self._ws.data_ptr(), self._ws.numel(), device=self.cache.device.index,
                         stream=stream_of(self.cache.device, stream))

    def free(self, slots: torch.Tensor, done: torch.Tensor | None = None, stream=None) -> None:
        """The listed rows become empty; pages that no row holds any more are free."""
        n = self._list(slots, "slots", done)
        if n:
            vkq.kv8_free(self.cache.struct, self.struct, slots.data_ptr(), n, _ptr(done), self._ws.data_ptr(),
                         self._ws.numel(), device=self.cache.device.index, stream=stream_of(self.cache.device, stream))

    def compact(self, used: torch.Tensor | None = None, stream=None) -> None:
        """The pages in use become pages 0 .. used - 1, their contents moved and the table renamed."""
        if used is not None:
            check_int32(used, (1,), "used", self.cache.device)
        vkq.kv8_compact(self.cache.struct, self.struct, _ptr(used), self._ws.data_ptr(), self._ws.numel(),
                        device=self.cache.device.index, stream=stream_of(self.cache.device, stream))
