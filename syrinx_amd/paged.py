"""A paged key/value cache on the GPU (libsxq sxq_kv_*): pages instead of max_seq positions a
stream, so that a server holds as many requests as their lengths allow.

``PagedKvCache`` owns the pools of every layer, the block tables, the lengths and the stack of
free pages.  One decode step of a batch is

    m = cache.reserve(add, capacity)                  # add: 0 or 1 a request; pages, slots, positions
    q = cache.append(layer, qkv, m, n_heads=..., rope=..., ...)   # per layer
    ctx = cache.attend(layer, q, rows=m.rows)

A query of ``attend`` sees every position of its request, those reserved together with it too:
right for the one new token of a decode step, and for the last of a prompt's tokens, not for the
tokens before it.  A map of several tokens a request (a prompt's) is for ``append``; a prompt's
tokens, each over its own prefix, are attended to by a paged engine (``DecoderLM.prefill``), and
of such a map ``attend`` takes the last token of each request, at m.cu[r + 1] - 1.

Nothing is copied to the host; every call enqueues on the current stream of the cache's device and
may be captured into a graph.  The reference keeps one growing tensor per stream
(KvCache, crates/syrinx-fish/src/s2/nn.rs:221-254); append is its QK-norm + RoPE + cache append
(nn.rs:325-339, crates/syrinx-lm/src/cv2/attention.rs:50-66) and attend its attention of one new
token (nn.rs:340-352).

The calls of one cache share its tables, and are ordered as the caller orders its streams.
"""
from __future__ import annotations

import ctypes
from dataclasses import dataclass
from typing import Optional

import torch

from ._lib import check, lib

RELEASE = -(1 << 31)  # an `add` that empties any request
_COUNTER_BYTES = 262144  # SXQ_KV_COUNTER_BYTES: the part of a workspace that starts as zeros

_DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 30}
_P = ctypes.c_void_p


class KvPages(ctypes.Structure):
    _fields_ = [("dtype", ctypes.c_int32), ("n_kv_heads", ctypes.c_int32), ("head_dim", ctypes.c_int32),
                ("page_size", ctypes.c_int32), ("n_pages", ctypes.c_int32), ("k", _P), ("v", _P),
                ("page_stride", ctypes.c_int64), ("head_stride", ctypes.c_int64), ("pos_stride", ctypes.c_int64)]


@dataclass
class SlotMap:
    """Where new tokens go: token t is at slot slots[t] and position pos[t] of request rows[t]
    (int32, -1 past the last token).  cu[r] is request r's first token, status[r] why it was
    refused (0: it was not; 1 out of pages, 2 longer than max_len's pages, 3 over the map's capacity)."""
    slots: torch.Tensor
    pos: torch.Tensor
    rows: torch.Tensor
    cu: Optional[torch.Tensor] = None
    status: Optional[torch.Tensor] = None


def _ptr(t):
    return t.data_ptr() if t is not None else None


# The current stream's handle without building a Stream object (2 us a call), where torch has it.
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


class PagedKvCache:
    """Keys and values of up to max_rows requests of up to max_len positions (rounded up to whole
    pages) in n_pages pages of page_size positions (a power of two, 16..1024).

    k, v: [n_layers, n_pages, n_kv_heads, page_size, head_dim]; table: int32 [max_rows, blocks];
    lens: int32 [max_rows]; free: int32 [n_pages], of which the first free_count[0] are free (to
    be written in place, never replaced)."""

    def __init__(self, n_layers, n_kv_heads, head_dim, *, n_pages, page_size=32, max_rows, max_len,
                 dtype=torch.bfloat16, device="cuda:0"):
        if dtype not in _DTYPES:
            raise ValueError(f"PagedKvCache: dtype {dtype} (float32, float16 or bfloat16)")
        if min(n_layers, max_rows, max_len) < 1:
            raise ValueError(f"PagedKvCache: {n_layers} layers, {max_rows} rows of {max_len} positions")
        device = torch.device(device)
        if device.type == "cuda" and device.index is None:
            device = torch.device("cuda", torch.cuda.current_device())
        self.device, self.dtype, self._index = device, dtype, device.index
        self.n_layers, self.n_kv_heads, self.head_dim = int(n_layers), int(n_kv_heads), int(head_dim)
        self.n_pages, self.page_size = int(n_pages), int(page_size)
        self.max_rows, self.max_len = int(max_rows), int(max_len)
        probe = self._pages(None, None)
        need = ctypes.c_size_t()
        check(lib().sxq_kv_attention_workspace(ctypes.byref(probe), 0, self.n_kv_heads, ctypes.byref(need)))
        if device.type != "cuda":
            raise ValueError(f"PagedKvCache: the cache lives on a GPU, not on {device}")
        self.max_blocks = -(-self.max_len // self.page_size)
        shape = (self.n_layers, self.n_pages, self.n_kv_heads, self.page_size, self.head_dim)
        self.k = torch.empty(shape, dtype=dtype, device=device)
        self.v = torch.empty(shape, dtype=dtype, device=device)
        self._layers = [self._pages(self.k[i], self.v[i]) for i in range(self.n_layers)]
        self._layer_refs = [ctypes.byref(p) for p in self._layers]
        self.table = torch.full((self.max_rows, self.max_blocks), -1, dtype=torch.int32, device=device)
        self.lens = torch.zeros(self.max_rows, dtype=torch.int32, device=device)
        # page 0 on top of the stack
        self.free = torch.arange(self.n_pages - 1, -1, -1, dtype=torch.int32, device=device)
        self.free_count = torch.full((1,), self.n_pages, dtype=torch.int32, device=device)
        self._need, self._ws = {}, {}

    def _pages(self, k, v):
        unit = self.head_dim * self.page_size
        return KvPages(_DTYPES[self.dtype], self.n_kv_heads, self.head_dim, self.page_size, self.n_pages, _ptr(k),
                       _ptr(v), unit * self.n_kv_heads, unit, self.head_dim)

    def _stream(self):
        return _raw_stream(self._index) if _raw_stream else torch.cuda.current_stream(self.device).cuda_stream

    def _layer(self, layer):
        if not 0 <= layer < self.n_layers:
            raise ValueError(f"PagedKvCache: layer {layer} of {self.n_layers}")
        return self._layer_refs[layer]

    def _want(self, what, t, dtype, numel=None):
        if (t.dtype is not dtype or t.device != self.device or not t.is_contiguous()
                or (numel is not None and t.numel() != numel)):
            size = f" of {numel} elements" if numel else ""
            raise ValueError(f"PagedKvCache: {what} must be a contiguous {dtype} tensor{size} on {self.device}, got "
                             f"{t.dtype} {tuple(t.shape)} on {t.device}")

    # -- pages ----------------------------------------------------------------------------
    def reserve(self, add, capacity=None, out: SlotMap = None) -> SlotMap:
        """Grow request r by add[r] tokens (add[r] < 0: shrink it; RELEASE empties it) and map
        the new tokens.  add: int32 [max_rows] on the GPU, or a sequence of ints (shorter: the
        rest 0; copied from the host, so not under capture).  capacity: the map's length (with
        a sequence: by default its tokens).  out: a map of an earlier call of this capacity, to
        write into.  Pages go to requests in order; a request that cannot get them stays as it
        was (status), and what it asked for counts against the requests after it: new prompts
        belong in the last rows, or in a call after the running requests' own."""
        if not torch.is_tensor(add):
            add = [int(a) for a in add]
            if len(add) > self.max_rows:
                raise ValueError(f"PagedKvCache.reserve: {len(add)} requests, {self.max_rows} rows")
            if capacity is None and out is None:
                capacity = sum(a for a in add if a > 0)
            add = torch.tensor(add + [0] * (self.max_rows - len(add)), dtype=torch.int32).to(self.device)
        self._want("add", add, torch.int32, self.max_rows)
        if out is None:
            if capacity is None:
                raise ValueError("PagedKvCache.reserve: a tensor of growths needs the map's capacity")
            cap, n = int(capacity), self.max_rows
            if cap < 0:
                raise ValueError(f"PagedKvCache.reserve: capacity {cap}")
            buf = torch.empty(3 * cap + 2 * n + 1, dtype=torch.int32, device=self.device)
            slots, pos, rows, cu, status = buf.split([cap, cap, cap, n + 1, n])
            out = SlotMap(slots, pos, rows, cu, status)
        else:
            cap = out.slots.numel()
            if capacity is not None and int(capacity) != cap:
                raise ValueError(f"PagedKvCache.reserve: capacity {capacity}, the map holds {cap}")
            for name, size in (("slots", cap), ("pos", cap), ("rows", cap), ("cu", self.max_rows + 1),
                               ("status", self.max_rows)):
                t = getattr(out, name)
                if t is None or t.numel() != size:
                    raise ValueError(f"PagedKvCache.reserve: out.{name} must hold {size} elements")
                self._want(f"out.{name}", t, torch.int32)
        check(lib().sxq_kv_reserve(self._index, self.page_size, self.n_pages, self.max_rows, self.max_blocks,
                                   add.data_ptr(), self.lens.data_ptr(), self.table.data_ptr(), self.max_blocks,
                                   self.free.data_ptr(), self.free_count.data_ptr(), cap, out.cu.data_ptr(),
                                   out.slots.data_ptr(), out.pos.data_ptr(), out.rows.data_ptr(), out.status.data_ptr(),
                                   self._stream()))
        return out

    # -- new tokens -----------------------------------------------------------------------
    def append(self, layer: int, qkv: torch.Tensor, slot_map: SlotMap, *, n_heads: int, q_norm=None, k_norm=None,
               eps: float = 1e-6, rope=None, interleaved=False, out: torch.Tensor = None) -> torch.Tensor:
        """The fused projection's rows qkv [T, (n_heads + 2 n_kv_heads) * head_dim] (f32, f16 or
        bf16; any row stride), token t to slot_map.slots[t]: QK-RMSNorm by q_norm / k_norm (f32
        [head_dim]) and RoPE by rope = (cos, sin) (f32 [positions, head_dim / 2]), keys and
        values into the layer's pages, the queries returned [T, n_heads * head_dim] in qkv's
        type.  A token without a slot leaves its row of out as it was."""
        hd, dev, dtype, shape = self.head_dim, self.device, qkv.dtype, qkv.shape
        width = (n_heads + 2 * self.n_kv_heads) * hd
        code = _DTYPES.get(dtype)
        if code is None or qkv.device != dev or len(shape) != 2 or shape[1] != width or qkv.stride(1) != 1:
            raise ValueError(f"PagedKvCache.append: qkv must be [T, {width}] f32, f16 or bf16 rows on {dev}, got "
                             f"{dtype} {tuple(shape)} on {qkv.device}")
        tokens = shape[0]
        stride = qkv.stride(0) if tokens > 1 else width
        if stride < width:
            raise ValueError(f"PagedKvCache.append: qkv's rows overlap (stride {stride}, width {width})")
        slots, pos = slot_map.slots, slot_map.pos
        self._want("slots", slots, torch.int32)
        self._want("pos", pos, torch.int32)
        if slots.numel() < tokens or pos.numel() < tokens:
            raise ValueError(f"PagedKvCache.append: {tokens} tokens, a map of {min(slots.numel(), pos.numel())}")
        qn = kn = cos = sin = None
        positions = 0
        if q_norm is not None:
            self._want("q_norm", q_norm, torch.float32, hd)
            qn = q_norm.data_ptr()
        if k_norm is not None:
            self._want("k_norm", k_norm, torch.float32, hd)
            kn = k_norm.data_ptr()
        if rope is not None:
            c, s = rope
            positions = c.shape[0]
            for name, t in (("cos", c), ("sin", s)):
                self._want(name, t, torch.float32, positions * (hd // 2))
                if t.dim() != 2 or t.shape[1] != hd // 2 or positions < 1:
                    raise ValueError(f"PagedKvCache.append: {name} must be [positions, {hd // 2}], got {tuple(t.shape)}")
            cos, sin = c.data_ptr(), s.data_ptr()
        if out is None:
            out = torch.empty((tokens, n_heads * hd), dtype=dtype, device=dev)
        else:
            self._want("out", out, dtype, tokens * n_heads * hd)
        check(lib().sxq_kv_append(self._index, self._layer(layer), code, qkv.data_ptr(), stride, tokens, n_heads, qn, kn,
                                  eps, cos, sin, positions, 1 if interleaved else 0, pos.data_ptr(), slots.data_ptr(),
                                  out.data_ptr(), self._stream()))
        return out

    # -- attention ------------------------------------------------------------------------
    def workspace(self, n_q: int, n_heads: int) -> torch.Tensor:
        """A workspace, ready for use, of attend over n_q queries of n_heads heads: one for every
        captured graph, kept while the graph lives."""
        need = self._need.get((n_q, n_heads))
        if need is None:
            size = ctypes.c_size_t()
            check(lib().sxq_kv_attention_workspace(self._layer_refs[0], n_q, n_heads, ctypes.byref(size)))
            need = self._need[(n_q, n_heads)] = int(size.value)
        ws = torch.empty(need, dtype=torch.uint8, device=self.device)
        ws[:_COUNTER_BYTES].zero_()
        return ws

    def _kept_workspace(self, n_q, n_heads):
        """Eager calls: one workspace per stream, kept.  Under capture: a fresh one, owned by
        the graph, its zeroing recorded."""
        if torch.cuda.current_device() == self._index:
            capturing = torch.cuda.is_current_stream_capturing()
        else:
            with torch.cuda.device(self._index):
                capturing = torch.cuda.is_current_stream_capturing()
        if capturing:
            return self.workspace(n_q, n_heads)
        stream = self._stream()
        ws = self._ws.get(stream)
        need = self._need.get((n_q, n_heads))
        if ws is None or need is None or ws.numel() < need:
            fresh = self.workspace(n_q, n_heads)
            if ws is None or ws.numel() < fresh.numel():
                ws = self._ws[stream] = fresh
        return ws

    def attend(self, layer: int, q: torch.Tensor, *, rows: torch.Tensor = None, scale: float = None,
               out: torch.Tensor = None, workspace: torch.Tensor = None) -> torch.Tensor:
        """softmax(scale q k^T) v of one new token per row of q [n, n_heads, head_dim] (or
        [n, n_heads * head_dim]) over the cache of request rows[n] (int32; None: request n) up to
        its length, whatever the query's own position: of several new tokens of a request only
        the last is attended as a decoder does.  q: the pages' type, or f32 over bf16 pages.  scale: 1 / sqrt(head_dim) by
        default.  A row of no request (rows[n] < 0) leaves out[n] as it was (without `out`:
        unset); an empty request gives zeros.  workspace: `workspace(n, n_heads)`, to keep its
        zeroing out of a captured graph."""
        hd, dev, dtype, shape = self.head_dim, self.device, q.dtype, q.shape
        code, dims = _DTYPES.get(dtype), len(shape)
        if code is None or q.device != dev or dims not in (2, 3) or (dims == 3 and shape[2] != hd):
            raise ValueError(f"PagedKvCache.attend: q must be [n, heads, {hd}] f32, f16 or bf16 on {dev}, got "
                             f"{dtype} {tuple(shape)} on {q.device}")
        n, width = shape[0], shape[1] * hd if dims == 3 else shape[1]
        if width == 0 or width % hd:
            raise ValueError(f"PagedKvCache.attend: q rows of {width} elements, heads of {hd}")
        n_heads = width // hd
        if out is None:
            out = torch.empty(shape, dtype=dtype, device=dev)
        elif out.device != dev or out.dtype is not dtype or out.shape != shape:
            raise ValueError(f"PagedKvCache.attend: out must be {dtype} {tuple(shape)} on {dev}")
        strides = []
        for what, t in (("q", q), ("out", out)):
            st = t.stride()
            if st[-1] != 1 or (dims == 3 and shape[1] > 1 and st[1] != hd):
                raise ValueError(f"PagedKvCache.attend: each row of {what} must be contiguous, got strides {st}")
            strides.append(st[0] if n > 1 else width)
        if rows is not None:
            self._want("rows", rows, torch.int32, n)
            rows = rows.data_ptr()
        if scale is None:
            scale = hd ** -0.5
        if n == 0:
            return out
        if workspace is None:
            workspace = self._kept_workspace(n, n_heads)
        else:
            self._want("workspace", workspace, torch.uint8)
        check(lib().sxq_kv_attention(self._index, self._layer(layer), code, q.data_ptr(), strides[0], n, n_heads, rows,
                                     self.lens.data_ptr(), self.max_rows, self.table.data_ptr(), self.max_blocks,
                                     self.max_blocks, scale, out.data_ptr(), strides[1], workspace.data_ptr(),
                                     workspace.numel(), self._stream()))
        return out
