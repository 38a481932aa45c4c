"""Serving many requests from one cache on gfx950: page tables, an 8-bit paged
KV cache, and attention over it, running on libloom_accel_amd.so.

=====================  ======================================================
``PageTable``          which pages of a pool each request holds, built on the
                       device from request lengths (``plan``, ``release``)
``StepPlan``           the rows of one step: row starts, positions, cache slots
``PagedCache``         keys and values as int8 codes, one scale for each page,
                       head and side (``append``, ``read``)
``attention``          causal grouped-query attention of a step's rows: decode
                       rows, chunks of prompts, or both in one call
=====================  ======================================================

The reference has no counterpart: its cache is one fp32 ring per layer and
sequence (poly/mha.go:95-96), which ``transformer.BitNetBlock.forward`` keeps.
``transformer.BitNetBlock.forward_paged`` runs a block on these operators.

A serving loop keeps the requests' lengths on the device and never waits:

    table = PageTable(requests, max_pages, num_pages, page_size=16)
    plan = table.plan(lens, new_tokens, rows)      # lens: before this step
    cache.append(k, v, plan.slots)                 # one cache per layer
    out = attention(q, cache, table.pages, plan.row_start, plan.positions)
    lens = plan.lens                               # lengths after it
    table.release(done)                            # uint8 flag per request

All calls run on the current stream of the tensors' device and allocate only
their outputs and workspaces, through torch, so they can be captured into
graphs.  There is no CPU or PyTorch fallback: a missing library raises.
"""
from __future__ import annotations

import ctypes as C
import functools

from . import _lib
from ._lib import check
from .bitnet import _torch

PAGE_SIZES = (16, 32, 64, 128)
HEAD_DIMS = (32, 64, 128, 256)


def _index(device) -> int:
    """Device number of an int or a torch device."""
    if isinstance(device, int):
        return device
    torch = _torch()
    d = torch.device(device)
    if d.type != "cuda":
        raise ValueError("the paged operators need a gfx950 device")
    return torch.cuda.current_device() if d.index is None else d.index


# (Host time counts here: a decode step's calls take the GPU 5 to 15 us each.
# Tensor.get_device and the raw device and stream getters are a fraction of the
# objects that Tensor.device and torch.cuda.current_device go through.)

def _device_of(t, what: str) -> int:
    dev = t.get_device()
    if dev < 0:
        raise ValueError(f"{what} must be a device tensor")
    return dev


def _want(t, dtype, shape, dev: int, what: str):
    """A contiguous tensor of this dtype, shape (None: any) and device."""
    if t.dtype is not dtype or t.get_device() != dev or not t.is_contiguous():
        raise ValueError(f"{what} must be a contiguous {str(dtype).split('.')[-1]} tensor on device {dev}")
    if shape is not None and t.shape != shape:
        raise ValueError(f"{what} is {tuple(t.shape)}, want {tuple(shape)}")
    return t.data_ptr()


def _call(dev: int, what: str, fn, *args) -> None:
    """fn(*args, stream) on device dev's current stream."""
    torch = _torch()
    if torch._C._cuda_getDevice() == dev:
        rc = fn(*args, torch._C._cuda_getCurrentRawStream(dev))
    else:
        with torch.cuda.device(dev):
            rc = fn(*args, torch._C._cuda_getCurrentRawStream(dev))
    if rc:
        check(rc, what)


def _rows_type() -> dict:
    torch = _torch()
    return {torch.float32: 0, torch.bfloat16: 1, torch.float64: 2}


@functools.lru_cache(maxsize=None)
def _row_type(dtype) -> int:
    t = _rows_type().get(dtype)
    if t is None:
        raise ValueError(f"rows of {dtype} are not supported")
    return t


def _row_stride(t, heads: int, hd: int, what: str) -> int:
    """Elements between rows of a rows x heads x hd tensor whose rows are dense."""
    s = t.stride()
    if (s[2] != 1 and hd > 1) or (s[1] != hd and heads > 1):
        raise ValueError(f"{what}: each row must be dense (heads x head_dim)")
    if t.shape[0] > 1 and s[0] < heads * hd:
        raise ValueError(f"{what}: rows must not overlap")
    return s[0]


class StepPlan:
    """The rows of one step, as ``PageTable.plan`` numbers them (int32 device
    tensors): ``row_start`` [requests + 1], ``lens`` [requests] with the new
    tokens, and for each row ``request``, ``positions`` and ``slots`` (-1 where
    a row has no place)."""

    __slots__ = ("row_start", "lens", "request", "positions", "slots", "_scratch")

    def __init__(self, row_start, lens, request, positions, slots, scratch=None):
        self.row_start = row_start
        self.lens = lens
        self.request = request
        self.positions = positions
        self.slots = slots
        self._scratch = scratch


class PageTable:
    """Tables of ``requests`` request slots, up to ``max_pages`` pages each,
    over a pool of ``num_pages`` pages of ``page_size`` tokens.

    ``pages`` [requests, max_pages], ``held`` [requests], ``free``
    [num_pages] and ``free_count`` [1] are int32 device tensors; the next page
    to give is ``free[free_count - 1]``."""

    def __init__(self, requests: int, max_pages: int, num_pages: int, page_size: int = 16, device=0):
        if page_size not in PAGE_SIZES:
            raise ValueError(f"page_size must be one of {PAGE_SIZES}")
        if requests <= 0 or max_pages <= 0 or num_pages <= 0:
            raise ValueError("requests, max_pages and num_pages must be positive")
        torch = _torch()
        self.requests, self.max_pages, self.num_pages, self.page_size = requests, max_pages, num_pages, page_size
        self.device = _index(device)
        kw = dict(dtype=torch.int32, device=f"cuda:{self.device}")
        self.pages = torch.empty(requests, max_pages, **kw)
        self.held = torch.empty(requests, **kw)
        self.free = torch.empty(num_pages, **kw)
        self.free_count = torch.empty(1, **kw)
        self._c = _lib.PageTable(self.pages.data_ptr(), self.held.data_ptr(), self.free.data_ptr(),
                                 self.free_count.data_ptr(), requests, max_pages, num_pages, page_size)
        self._p = C.byref(self._c)
        self.reset()

    def reset(self) -> None:
        """Every page free, no request holds any."""
        _call(self.device, "page_table_reset", _lib.lib().loom_amd_page_table_reset, self._p)

    def plan(self, lens, new_tokens, rows: int) -> StepPlan:
        """Rows and slots of a step that appends new_tokens[r] tokens to
        request r, which has lens[r] (int32 device tensors).  rows is the
        capacity of the row outputs, at least the sum of new_tokens; rows
        behind the last are -1.  Requests take the pages they lack; one whose
        pages, table or rows do not suffice gets none, keeps its length
        (``plan.lens``), and its rows are -1."""
        torch = _torch()
        n = self.requests
        dev = self.device
        pl = _want(lens, torch.int32, (n,), dev, "lens")
        pn = _want(new_tokens, torch.int32, (n,), dev, "new_tokens")
        if rows < 0:
            raise ValueError("rows must not be negative")
        buf = torch.empty(6 * n + 1 + 3 * rows, dtype=torch.int32, device=lens.device)
        scratch, start, after, req, pos, slots = buf.split_with_sizes((4 * n, n + 1, n, rows, rows, rows))
        at = buf.data_ptr()
        at1 = at + 16 * n
        at2 = at1 + 4 * n + 4
        at3 = at2 + 4 * n
        c = _lib.PagePlan(at1, at2, at3, at3 + 4 * rows, at3 + 8 * rows, at)
        _call(dev, "page_table_plan", _lib.lib().loom_amd_page_table_plan, self._p, pl, pn, rows, C.byref(c))
        return StepPlan(start, after, req, pos, slots, scratch)

    def release(self, done) -> None:
        """Gives back the pages of every request whose flag (uint8 or bool
        device tensor, one per request) is set."""
        torch = _torch()
        if done.dtype == torch.bool:
            done = done.view(torch.uint8)
        p = _want(done, torch.uint8, (self.requests,), self.device, "done")
        _call(self.device, "page_table_release", _lib.lib().loom_amd_page_table_release, self._p, p)


class PagedCache:
    """Keys and values of one layer as int8 codes in pages, with an fp32 scale
    for each page, head and side (value = code * scale).  2 bytes per cached key
    and value where the fp32 ring takes 8.

    The codes lie in blocks of 16 tokens, in the order of attention's matrix
    operands:

        k [num_pages, kv_heads, page_size / 16, head_dim / 16, 16 tokens, 16]
        v [num_pages, kv_heads, page_size / 16, head_dim, 16 tokens]
        k_scale, v_scale [num_pages, kv_heads]

    ``from_tensors`` and ``codes`` convert from and to plain order."""

    def __init__(self, num_pages: int, page_size: int, kv_heads: int, head_dim: int, device=0):
        torch = _torch()
        self._shape(num_pages, page_size, kv_heads, head_dim, _index(device))
        kw = dict(device=f"cuda:{self.device}")
        b = page_size // 16
        self._hold(torch.zeros(num_pages, kv_heads, b, head_dim // 16, 16, 16, dtype=torch.int8, **kw),
                   torch.zeros(num_pages, kv_heads, b, head_dim, 16, dtype=torch.int8, **kw),
                   torch.zeros(num_pages, kv_heads, dtype=torch.float32, **kw),
                   torch.zeros(num_pages, kv_heads, dtype=torch.float32, **kw))

    @classmethod
    def from_tensors(cls, k, v, k_scale, v_scale) -> "PagedCache":
        """A cache that holds these codes and scales: k int8 [num_pages,
        kv_heads, page_size, head_dim], v int8 [num_pages, kv_heads, head_dim,
        page_size], scales float32 [num_pages, kv_heads], none negative.  They
        are copied."""
        torch = _torch()
        if k.dim() != 4:
            raise ValueError("k must be [num_pages, kv_heads, page_size, head_dim]")
        pages, heads, page, hd = k.shape
        self = cls.__new__(cls)
        dev = _device_of(k, "k")
        self._shape(pages, page, heads, hd, dev)
        _want(k, torch.int8, None, dev, "k")
        _want(v, torch.int8, (pages, heads, hd, page), dev, "v")
        _want(k_scale, torch.float32, (pages, heads), dev, "k_scale")
        _want(v_scale, torch.float32, (pages, heads), dev, "v_scale")
        fmt = torch.contiguous_format
        self._hold(k.view(pages, heads, page // 16, 16, hd // 16, 16).permute(0, 1, 2, 4, 3, 5).clone(memory_format=fmt),
                   v.view(pages, heads, hd, page // 16, 16).permute(0, 1, 3, 2, 4).clone(memory_format=fmt),
                   k_scale.clone(), v_scale.clone())
        return self

    def codes(self):
        """(k, v): copies of the codes, both int8 [num_pages, kv_heads,
        page_size, head_dim]."""
        shape = (self.num_pages, self.kv_heads, self.page_size, self.head_dim)
        return (self.k.permute(0, 1, 2, 4, 3, 5).reshape(shape), self.v.transpose(3, 4).reshape(shape))

    def _shape(self, pages: int, page: int, heads: int, hd: int, dev: int) -> None:
        if page not in PAGE_SIZES:
            raise ValueError(f"page_size must be one of {PAGE_SIZES}")
        if hd not in HEAD_DIMS:
            raise ValueError(f"head_dim must be one of {HEAD_DIMS}")
        if pages <= 0 or heads <= 0 or pages * page > 2 ** 31 - 1:
            raise ValueError("a cache holds 1 to 2^31 - 1 tokens of at least one head")
        self.num_pages, self.kv_heads, self.page_size, self.head_dim = pages, heads, page, hd
        self.device = dev

    def _hold(self, k, v, k_scale, v_scale) -> None:
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self._c = _lib.KvPages(*(t.data_ptr() for t in (k, v, k_scale, v_scale)), self.num_pages, self.page_size,
                               self.kv_heads, self.head_dim)
        self._p = C.byref(self._c)

    def append(self, k, v, slots) -> None:
        """Quantizes rows of keys and values ([rows, kv_heads, head_dim],
        float32 or bfloat16, rows dense, any row stride) into their slots
        (int32 [rows], as a plan numbers them; -1 skips a row)."""
        torch = _torch()
        shape = (slots.shape[0], self.kv_heads, self.head_dim)
        if k.shape != shape or v.shape != shape:
            raise ValueError(f"k is {tuple(k.shape)} and v {tuple(v.shape)}, want {shape}")
        if k.dtype != v.dtype or k.dtype not in (torch.float32, torch.bfloat16):
            raise ValueError("k and v must both be float32 or both bfloat16")
        if _device_of(k, "k") != self.device or _device_of(v, "v") != self.device:
            raise ValueError(f"k and v must be on device {self.device}")
        ps = _want(slots, torch.int32, None, self.device, "slots")
        _call(self.device, "kv_append", _lib.lib().loom_amd_kv_append, self._p, k.data_ptr(), v.data_ptr(),
              _row_type(k.dtype), shape[0], _row_stride(k, shape[1], shape[2], "k"),
              _row_stride(v, shape[1], shape[2], "v"), ps)

    def read(self, slots):
        """(k, v) values of slots (int32 [rows]) as float32 [rows, kv_heads,
        head_dim]; zeros for a slot of -1."""
        torch = _torch()
        ps = _want(slots, torch.int32, None, self.device, "slots")
        if slots.dim() != 1:
            raise ValueError("slots must be one-dimensional")
        n = slots.shape[0]
        k = torch.empty(n, self.kv_heads, self.head_dim, dtype=torch.float32, device=slots.device)
        v = torch.empty_like(k)
        _call(self.device, "kv_read", _lib.lib().loom_amd_kv_read, self._p, ps, n, k.data_ptr(), v.data_ptr())
        return k, v


_workspaces: dict = {}


def _attention_workspace(*shape) -> int:
    """Bytes of workspace for (rows, heads, kv_heads, head_dim, requests, max_context)."""
    need = _workspaces.get(shape)
    if need is None:
        n = C.c_size_t()
        check(_lib.lib().loom_amd_paged_attention_workspace(*shape, C.byref(n)), "paged_attention")
        if len(_workspaces) >= 4096:
            _workspaces.clear()
        need = _workspaces[shape] = n.value
    return need


def attention(q, cache: PagedCache, pages, row_start, positions, scale: float | None = None,
              max_context: int | None = None, out=None):
    """Causal attention of rows q [rows, heads, head_dim] (float32, bfloat16 or
    float64, rows dense, any row stride) over the cache; returns out, like q.

    pages [requests, max_pages], row_start [requests + 1] and positions [rows]
    are int32 device tensors (``PageTable.pages`` and a ``StepPlan``'s): row t
    of request r attends to positions 0 .. positions[t] of r's pages.  heads is
    a multiple of the cache's key/value heads.  scale defaults to 1 /
    sqrt(head_dim).  max_context (default: all of the table) promises that no
    position is past it, so that fewer workgroups are launched.  A row with
    position -1 gives zeros; rows of no request keep what out held."""
    torch = _torch()
    if q.dim() != 3 or q.shape[2] != cache.head_dim or q.shape[1] == 0 or q.shape[1] % cache.kv_heads:
        raise ValueError(f"q is {tuple(q.shape)}, want [rows, a multiple of {cache.kv_heads} heads, "
                         f"{cache.head_dim}]")
    rows, heads, hd = q.shape
    dev = cache.device
    if _device_of(q, "q") != dev:
        raise ValueError(f"q must be on device {dev}")
    kind = _row_type(q.dtype)
    if pages.dim() != 2:
        raise ValueError("pages must be [requests, max_pages]")
    requests, max_pages = pages.shape
    if requests == 0 or max_pages == 0:
        raise ValueError("pages must hold at least one request and one page")
    pp = _want(pages, torch.int32, None, dev, "pages")
    pr = _want(row_start, torch.int32, (requests + 1,), dev, "row_start")
    po = _want(positions, torch.int32, (rows,), dev, "positions")
    if max_context is None:
        max_context = max_pages * cache.page_size
    elif not 0 <= max_context <= max_pages * cache.page_size:
        raise ValueError("max_context must be within the table")
    q_stride = _row_stride(q, heads, hd, "q")
    if out is None:
        out = torch.empty(rows, heads, hd, dtype=q.dtype, device=q.device)
    elif out.shape != q.shape or out.dtype != q.dtype or out.device != q.device:
        raise ValueError("out must have q's shape, dtype and device")
    out_stride = _row_stride(out, heads, hd, "out")
    need = _attention_workspace(rows, heads, cache.kv_heads, hd, requests, max_context)
    ws = torch.empty(need, dtype=torch.uint8, device=q.device) if need else None
    _call(dev, "paged_attention", _lib.lib().loom_amd_paged_attention, cache._p, pp, requests, max_pages, pr, po,
          q.data_ptr(), kind, rows, heads, q_stride, hd ** -0.5 if scale is None else float(scale), max_context,
          out.data_ptr(), out_stride, ws.data_ptr() if need else None, need)
    return out


__all__ = ["PageTable", "StepPlan", "PagedCache", "attention", "PAGE_SIZES", "HEAD_DIMS"]
