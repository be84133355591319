"""The paged 4-bit key/value cache of an attention layer, and the attention
over it: the gofann_kv_* C ABI over torch device tensors (torch holds device
memory only; every computation is a HIP kernel of libgofann_hip.so).

A decoding step of a long-context model is a search of the cached keys by the
step's queries.  The cache holds keys and values in 4 bits; `append` writes a
step's tokens; `attend` reads every position, or those that a filter's bits
leave; `select` scores the pages' boxes by integer products and names the few
blocks that each token and key/value head should read, and `attend` with
those reads nothing else.  The reference has no counterpart.

    cache = KvCache.empty(ctx, pages=4096, kv_heads=8, dim=128)
    batch = KvBatch(page_table, lengths, max_length=131072)     # one token each
    cache.append(batch, k, v)
    out = cache.attend(batch, q)                                 # all positions
    out = cache.attend(batch, q, blocks=cache.select(batch, q, 64))

Calls are asynchronous on the context's stream, which has to be torch's
current one, on the context's device.  Everything may be captured in a graph
once a call of the same sizes has run.  The graph then uses the context's
scratch: order its replays with each other and with the context's other calls,
as work on one stream is.
"""
from __future__ import annotations

import ctypes as C

import torch

from . import _lib

_ELEM = {torch.bfloat16: _lib.ELEM_BF16, torch.float16: _lib.ELEM_F16}
# The handle of torch's current stream, as torch.cuda.current_stream(i).cuda_stream.
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or \
    (lambda i: torch.cuda.current_stream(i).cuda_stream)
_current_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device
DIMS = (64, 128, 256)
PAGE_SIZES = (32, 64, 128, 256)


def _shapes(pages: int, heads: int, page: int, dim: int) -> dict:
    return dict(k_codes=(pages, heads, page, dim // 2), k_scales=(pages, heads, page, dim // 32),
                v_codes=(pages, heads, page // 8, 16, 8, dim // 32),
                v_scales=(pages, heads, page // 8, dim // 32, 8),
                box=(pages, heads, 2, dim), box_scale=(pages, heads))


def _counts(**kw: int) -> None:
    for name, n in kw.items():
        if not 0 <= n < 1 << 32:
            raise ValueError(f"{name} must be in [0, 2^32)")


class KvBatch:
    """The sequences of one call (gofann_kv_batch).

    page_table [sequences][width] i32: the page of each block of a sequence,
    outside [0, pages) where there is none; lengths [sequences] i32, this
    call's tokens among them; query_offsets [sequences + 1] i32: the first row
    of each sequence's tokens, which are its last positions (None: one token
    each); visible [sequences][words] i32: bit t % 32 of word t / 32 says
    whether position t may be attended to (None: all).

    The tensors are read when a call runs on the device, so they may be
    updated in place between calls; `queries`, `max_queries` and `max_length`
    are the host's bounds for the launches: rows in all, at least the tokens
    of any sequence, at least any length.
    """

    def __init__(self, page_table: torch.Tensor, lengths: torch.Tensor,
                 query_offsets: torch.Tensor | None = None, *, queries: int | None = None,
                 max_queries: int | None = None, max_length: int,
                 visible: torch.Tensor | None = None):
        if page_table.dim() != 2 or lengths.dim() != 1 or lengths.shape[0] != page_table.shape[0]:
            raise ValueError("page_table is [sequences][width] and lengths [sequences]")
        n = lengths.shape[0]
        if query_offsets is None:
            if queries not in (None, n) or max_queries not in (None, 1):
                raise ValueError("without query_offsets there is one token a sequence")
            queries, max_queries = n, 1
        elif query_offsets.shape != (n + 1,):
            raise ValueError("query_offsets is [sequences + 1]")
        elif queries is None or max_queries is None:
            raise ValueError("query_offsets needs queries and max_queries")
        _counts(queries=queries, max_queries=max_queries, max_length=max_length)
        if visible is not None and (visible.dim() != 2 or visible.shape[0] != n):
            raise ValueError("visible is [sequences][words]")
        for name, t in (("page_table", page_table), ("lengths", lengths),
                        ("query_offsets", query_offsets), ("visible", visible)):
            if t is None:
                continue
            if t.dtype != torch.int32:
                raise ValueError(f"{name} must be int32")
            if t.device != page_table.device:
                raise ValueError(f"{name} is on another device")
            if t.numel() and t.stride(-1) != 1:
                raise ValueError(f"{name} must be contiguous along its last axis")
        self.device = page_table.device
        self.queries, self.max_queries, self.max_length = queries, max_queries, max_length
        self.sequences = n
        self._keep = (page_table, lengths, query_offsets, visible)
        stride = lambda t: max(t.stride(0), t.shape[1]) if t.shape[0] > 1 else t.shape[1]  # noqa: E731
        for name, t in (("page_table", page_table), ("visible", visible)):
            if t is not None and t.shape[0] > 1 and t.stride(0) < t.shape[1]:
                raise ValueError(f"rows of {name} overlap")
        self.view = _lib.KvBatchView(
            page_table.data_ptr(), lengths.data_ptr(), _lib.ptr(query_offsets), _lib.ptr(visible),
            n, page_table.shape[1], stride(page_table), 0 if visible is None else stride(visible),
            queries, max_queries, max_length)
        if visible is not None:
            self.view.visible_width = visible.shape[1]
            if visible.shape[1] == 0:
                # Nothing is visible, where NULL would be everything; the
                # address is not read.
                self.view.visible, self.view.visible_stride = lengths.data_ptr(), 0


class KvCache:
    """The cache's arrays (gofann_kv_cache) and the calls on them.

    k_codes [pages][kv_heads][page][dim/2], k_scales [..][page][dim/32],
    v_codes [..][page/8][16][8][dim/32], v_scales [..][page/8][dim/32][8], all
    u8, and, for `select`, box [..][2][dim] i8 and box_scale [pages][kv_heads]
    u8.  dtype: of queries, keys, values and outputs.
    """

    def __init__(self, ctx: _lib.Context, k_codes: torch.Tensor, k_scales: torch.Tensor,
                 v_codes: torch.Tensor, v_scales: torch.Tensor, *, box: torch.Tensor | None = None,
                 box_scale: torch.Tensor | None = None, dtype: torch.dtype = torch.bfloat16):
        if dtype not in _ELEM:
            raise ValueError("dtype must be bfloat16 or float16")
        if k_codes.dim() != 4:
            raise ValueError("k_codes is [pages][kv_heads][page][dim/2]")
        pages, heads, page, half = k_codes.shape
        dim = 2 * half
        if dim not in DIMS or page not in PAGE_SIZES:
            raise ValueError(f"dim must be one of {DIMS} and page one of {PAGE_SIZES}")
        if (box is None) != (box_scale is None):
            raise ValueError("box and box_scale come together")
        arrays = dict(k_codes=k_codes, k_scales=k_scales, v_codes=v_codes, v_scales=v_scales)
        if box is not None:
            arrays.update(box=box, box_scale=box_scale)
        shapes = _shapes(pages, heads, page, dim)
        for name, t in arrays.items():
            if tuple(t.shape) != shapes[name]:
                raise ValueError(f"{name} must be {shapes[name]}, got {tuple(t.shape)}")
            if t.dtype != (torch.int8 if name == "box" else torch.uint8):
                raise ValueError(f"{name} has the wrong type")
            if not t.is_contiguous() or t.device != k_codes.device:
                raise ValueError(f"{name} must be contiguous and on one device with k_codes")
        self.ctx, self.lib = ctx, ctx.lib
        self.dtype, self.device = dtype, k_codes.device
        self._index = k_codes.device.index if k_codes.device.type == "cuda" else -1
        self.pages, self.kv_heads, self.page, self.dim = pages, heads, page, dim
        self.__dict__.update(arrays)
        self.boxed = box is not None
        self.view = _lib.KvCacheView(k_codes.data_ptr(), k_scales.data_ptr(), v_codes.data_ptr(),
                                     v_scales.data_ptr(), _lib.ptr(box), _lib.ptr(box_scale),
                                     pages, heads, page, dim, _ELEM[dtype])

    @classmethod
    def empty(cls, ctx: _lib.Context, *, pages: int, kv_heads: int, dim: int, page: int = 64,
              dtype: torch.dtype = torch.bfloat16, boxes: bool = True) -> "KvCache":
        """A cache of unwritten pages on the context's device."""
        if dim not in DIMS or page not in PAGE_SIZES:
            raise ValueError(f"dim must be one of {DIMS} and page one of {PAGE_SIZES}")
        shapes = _shapes(pages, kv_heads, page, dim)
        new = {n: torch.empty(s, dtype=torch.int8 if n == "box" else torch.uint8,
                              device=torch.device("cuda", ctx.device))
               for n, s in shapes.items() if boxes or not n.startswith("box")}
        return cls(ctx, **new, dtype=dtype)

    # -- checks ----------------------------------------------------------
    def _rows(self, name: str, t: torch.Tensor, queries: int, heads: int | None,
              written: bool = False) -> _lib.KvRows:
        shape = t.shape
        if shape == (queries, heads, self.dim) and t.dtype is self.dtype and \
                t.is_contiguous() and t.device == self.device:
            return _lib.KvRows(t.data_ptr(), heads * self.dim, self.dim)
        st, sh, sd = t.stride() if t.dim() == 3 else (0, 0, 0)
        if len(shape) != 3 or shape[0] != queries or shape[2] != self.dim or \
                (heads is not None and shape[1] != heads):
            raise ValueError(f"{name} must be [{queries}][{heads if heads is not None else 'heads'}]"
                             f"[{self.dim}], got {tuple(shape)}")
        if t.dtype != self.dtype or t.device != self.device:
            raise ValueError(f"{name} must be {self.dtype} on {self.device}")
        if sd != 1:
            raise ValueError(f"{name} must be contiguous along its channels")
        if written and ((shape[0] > 1 and st < self.dim) or (shape[1] > 1 and sh < self.dim)
                        or (shape[0] > 1 and shape[1] > 1 and st < sh * shape[1]
                            and sh < st * shape[0])):
            raise ValueError(f"rows of {name} overlap")
        return _lib.KvRows(t.data_ptr(), st, sh)

    def _ready(self, batch: KvBatch) -> None:
        if batch.device != self.device:
            raise ValueError("the batch is on another device")
        if self._index != self.ctx.device:
            raise ValueError("the cache is not on the context's device")
        if _current_device() != self._index:
            raise _lib.GofannError("torch's current device is not the context's")
        if _raw_stream(self._index) != self.ctx.stream:
            raise _lib.GofannError("the context is bound to another stream than torch's current "
                                   "one: call ctx.bind_stream")

    # -- calls -----------------------------------------------------------
    def append(self, batch: KvBatch, k: torch.Tensor, v: torch.Tensor, *,
               k_held: torch.Tensor | None = None, v_held: torch.Tensor | None = None) -> None:
        """Quantizes keys and values [queries][kv_heads][dim] of the batch's
        tokens into their pages, and renews those pages' boxes.  k_held and
        v_held, of the same shape, get the values that the cache then holds
        (what later steps will see); rows of tokens without a page keep
        theirs."""
        self._ready(batch)
        n, h = batch.queries, self.kv_heads
        rk, rv = self._rows("k", k, n, h), self._rows("v", v, n, h)
        hk = None if k_held is None else self._rows("k_held", k_held, n, h, True)
        hv = None if v_held is None else self._rows("v_held", v_held, n, h, True)
        self.ctx.check(self.lib.gofann_kv_append(self.ctx.handle, self.view, batch.view, rk, rv, hk, hv))

    def select(self, batch: KvBatch, q: torch.Tensor, width: int, *, first: int = 1, last: int = 2,
               out: torch.Tensor | None = None) -> torch.Tensor:
        """Blocks [queries][kv_heads][width] i32 for each token to read,
        ascending, -1 past the last: its sequence's `first` first and `last`
        last ones, then those whose boxes score highest against any of the
        group's queries."""
        self._ready(batch)
        _counts(width=width, first=first, last=last)
        rq = self._rows("q", q, batch.queries, q.shape[1] if q.dim() == 3 else None)
        shape = (batch.queries, self.kv_heads, width)
        if out is None:
            out = torch.empty(shape, dtype=torch.int32, device=self.device)
        elif out.shape != shape or out.dtype != torch.int32 or out.device != self.device or \
                not out.is_contiguous():
            raise ValueError(f"out must be contiguous int32 {shape}")
        self.ctx.check(self.lib.gofann_kv_select(self.ctx.handle, self.view, batch.view, rq,
                                                 q.shape[1], width, first, last, out.data_ptr()))
        return out

    def attend(self, batch: KvBatch, q: torch.Tensor, *, scale: float | None = None,
               blocks: torch.Tensor | None = None, out: torch.Tensor | None = None,
               lse: torch.Tensor | None = None) -> torch.Tensor:
        """softmax(scale q.k) v of queries [queries][heads][dim] over the
        positions up to each token's own that the filter leaves, or of these
        only the ones in `blocks` (as `select` gives them).  scale: dim ** -0.5
        by default.  lse [queries][heads] f32 gets the log of the sums of
        exponentials.  A row with nothing to read is zero (lse -inf)."""
        self._ready(batch)
        heads = q.shape[1] if q.dim() == 3 else None
        rq = self._rows("q", q, batch.queries, heads)
        if out is None:
            out = torch.empty_like(q, memory_format=torch.contiguous_format)
            ro = _lib.KvRows(out.data_ptr(), heads * self.dim, self.dim)
        else:
            ro = self._rows("out", out, batch.queries, heads, True)
        width = 0
        if blocks is not None:
            if blocks.dim() != 3 or blocks.shape[:2] != (batch.queries, self.kv_heads) or \
                    blocks.dtype != torch.int32 or blocks.device != self.device or \
                    not blocks.is_contiguous():
                raise ValueError("blocks must be contiguous int32 [queries][kv_heads][width]")
            width = blocks.shape[2]
        if lse is not None and (lse.shape != (batch.queries, heads) or lse.dtype != torch.float32
                                or lse.device != self.device or not lse.is_contiguous()):
            raise ValueError("lse must be contiguous float32 [queries][heads]")
        self.ctx.check(self.lib.gofann_kv_attention(
            self.ctx.handle, self.view, batch.view, rq, heads,
            self.dim ** -0.5 if scale is None else scale, _lib.ptr(blocks), width, ro, _lib.ptr(lse)))
        return out
