"""Drafted tokens over a K/V cache in pages: the operators of one step of drafted decoding on torch tensors.

    pool = PagePool.create(n_pages, page_size, batch, max_pages)       # tables and the stack of free pages
    cache = PagedCache.empty(layers, n_pages, heads, page_size, head_dim)
    plan = pool.plan(kept, fresh, rows, parents)                       # pages, slots, positions, masks, work units
    for i in range(layers):
        layer = cache.layer(i)
        write(layer, k, v, plan.slots)
        out = tree_attention(q, layer, pool.table, kept, plan.row_start, plan.units, plan.unit_start, nodes, mask=plan.mask)
    best, path, count, tokens = accept(logits, drafted, parents, plan.row_start, nodes)
    compact(cache, pool.table, kept, path, count)
    pool.commit(plan); kept += count

Thin wrappers over the C ABI (``mw_paged_*``, ``mw_tree_*`` in include/mwhip.h, where the semantics stand).  Tensors are
device tensors of one GPU; the launches go to torch's current stream of that GPU and the calls return at once, so they order
like torch's own operators and can be captured into a graph.  Outputs and workspaces come from torch's allocator; nothing
is kept between calls.  There is no backward pass.  A bad argument raises ``EngineError``.
"""
from __future__ import annotations

import ctypes as C
import math
from typing import Optional

import torch

from . import _lib
from .engine import EngineError

_FLOATS = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
_CODES = (torch.uint8, torch.float8_e4m3fn)
_E4M3 = 3
_INT = torch.int32


def _fail(what: str):
    raise EngineError(what)


def _check(rc: int, what: str):
    if rc != 0:
        raise EngineError(f"{what} failed ({rc}): {_lib.load().mw_last_error(None).decode()}")


def _stream(device: int) -> int:
    return torch.cuda.current_stream(device).cuda_stream


def _array(t, name: str, dtype, shape, device: int) -> int:
    """Address of a contiguous tensor of the expected type, shape (None: any extent) and GPU."""
    if t.dtype is not dtype or t.dim() != len(shape) or not t.is_contiguous():
        _fail(f"{name} must be a contiguous {dtype} tensor of {len(shape)} dimensions, got {t.dtype} {tuple(t.shape)}")
    for have, want in zip(t.shape, shape):
        if want is not None and have != want:
            _fail(f"{name} must have shape {tuple(shape)}, got {tuple(t.shape)}")
    if t.get_device() != device:
        _fail(f"{name} must be on cuda:{device}, got {t.device}")
    return t.data_ptr()


def _gpu_of(t, name: str) -> int:
    if not t.is_cuda:
        _fail(f"{name} must be on a GPU, got {t.device}")
    return t.get_device()


def _rows3(t, name: str, device: int):
    """(address, row stride, head stride) of a [rows, heads, head_dim] tensor whose last dimension is dense."""
    if t.dim() != 3 or (t.stride(2) != 1 and t.shape[2] > 1):
        _fail(f"{name} must be [rows, heads, head_dim] with dense rows, got {tuple(t.shape)} strides {t.stride()}")
    if t.requires_grad:
        _fail(f"{name} requires a gradient, and there is no backward pass")
    if t.get_device() != device:
        _fail(f"{name} must be on cuda:{device}, got {t.device}")
    return t.data_ptr(), t.stride(0), t.stride(1)


class PagedCache:
    """K/V in pages: ``k``, ``v`` [layers, pages, heads, page_size, head_dim] (or without the layers: one layer) of float16 or
    bfloat16, or e4m3 codes (uint8 / float8_e4m3fn) with the row scales ``k_scale``, ``v_scale`` (float32, contiguous, the
    shape without head_dim).  The order of pages, heads and tokens in memory is free (transposed views are fine); rows are
    dense and start at multiples of 16 bytes.  ``page_size``: a power of two in 16..4096; ``head_dim``: 64 or 128."""

    def __init__(self, k, v, k_scale=None, v_scale=None):
        if k.dim() not in (4, 5) or k.shape != v.shape or k.dtype != v.dtype or k.stride() != v.stride():
            _fail(f"k and v must be [(layers,) pages, heads, page_size, head_dim] of one type and layout, got {tuple(k.shape)} {k.dtype} "
                  f"and {tuple(v.shape)} {v.dtype}")
        self.device = _gpu_of(k, "k")
        codes = k.dtype in _CODES
        if not codes and k.dtype not in (torch.float16, torch.bfloat16):
            _fail(f"a cache holds float16, bfloat16 or e4m3 codes, got {k.dtype}")
        if k.stride(-1) != 1 or v.get_device() != self.device:
            _fail("rows of the cache must be dense, and k and v on one GPU")
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self.layers = k.shape[0] if k.dim() == 5 else None
        n_pages, heads, page, dim = k.shape[-4:]
        ks = vs = None
        if codes:
            if k_scale is None or v_scale is None:
                _fail("an e4m3 cache needs its row scales")
            ks = _array(k_scale, "k_scale", torch.float32, k.shape[:-1], self.device)
            vs = _array(v_scale, "v_scale", torch.float32, k.shape[:-1], self.device)
        elif k_scale is not None or v_scale is not None:
            _fail("row scales belong to an e4m3 cache")
        self.dtype = _E4M3 if codes else _FLOATS[k.dtype]
        self.page_size, self.heads, self.head_dim, self.n_pages = page, heads, dim, n_pages
        self.struct = _lib.PagedCache(k.data_ptr(), v.data_ptr(), ks, vs, k.stride(-4), k.stride(-3), k.stride(-2), n_pages, page, heads, dim,
                                      self.dtype)

    @classmethod
    def empty(cls, layers: int, n_pages: int, heads: int, page_size: int, head_dim: int, dtype=torch.float16, device="cuda") -> "PagedCache":
        """A cache of its own memory; ``dtype`` float16, bfloat16 or float8_e4m3fn.  The rows hold nothing yet."""
        shape = (layers, n_pages, heads, page_size, head_dim)
        if dtype in _CODES:
            s = [torch.zeros(shape[:-1], dtype=torch.float32, device=device) for _ in range(2)]
            return cls(torch.zeros(shape, dtype=torch.uint8, device=device), torch.zeros(shape, dtype=torch.uint8, device=device), *s)
        return cls(torch.zeros(shape, dtype=dtype, device=device), torch.zeros(shape, dtype=dtype, device=device))

    def layer(self, i: int) -> "PagedCache":
        """Layer ``i`` as a cache of one layer (a view)."""
        if self.layers is None:
            _fail("this cache is one layer")
        scales = (None, None) if self.k_scale is None else (self.k_scale[i], self.v_scale[i])
        return PagedCache(self.k[i], self.v[i], *scales)

    def _one(self) -> "PagedCache":
        if self.layers is not None:
            _fail("this call takes one layer of a cache: cache.layer(i)")
        return self


class StepPlan:
    """What ``PagePool.plan`` made: row_start [batch + 1], slots (int64) and positions [rows], mask [rows, words] (None: chains),
    admitted, pages [batch], n_free [1], units [batch + chunks, 4], unit_start [batch + 1]; int32, views of one buffer."""

    _NAMES = ("units", "slots", "row_start", "admitted", "pages", "n_free", "unit_start", "positions", "mask")

    def __init__(self, batch: int, rows: int, words: int, n_units: int, device):
        self.batch, self.rows, self.words, self.n_units = batch, rows, words, n_units
        self._sizes = (4 * n_units, 2 * rows, batch + 1, batch, batch, 1, batch + 1, rows, rows * words)
        self._buf = torch.empty(sum(self._sizes), dtype=_INT, device=device)
        self._parts = None

    def _addresses(self):
        at, out = self._buf.data_ptr(), []
        for n in self._sizes:
            out.append(at)
            at += 4 * n
        return out

    def __getattr__(self, name: str):            # the views are made when the first one is asked for
        if name not in self._NAMES:
            raise AttributeError(name)
        if self._parts is None:
            p = dict(zip(self._NAMES, self._buf.split(self._sizes)))
            p["units"], p["slots"] = p["units"].view(self.n_units, 4), p["slots"].view(torch.int64)
            p["mask"] = p["mask"].view(self.rows, self.words) if self.words else None
            self._parts = p
        return self._parts[name]


class PagePool:
    """Tables [batch, max_pages], pages held per request [batch] and the stack of free pages [n_pages] with its height [1]."""

    def __init__(self, table, pages, free, n_free, page_size: int):
        self.device = _gpu_of(table, "table")
        if table.dim() != 2 or table.dtype is not _INT or table.stride(1) != 1:
            _fail(f"table must be int32 [batch, max_pages] with dense rows, got {table.dtype} {tuple(table.shape)}")
        self.batch, self.max_pages = table.shape
        _array(pages, "pages", _INT, (self.batch,), self.device)
        _array(free, "free", _INT, (None,), self.device)
        _array(n_free, "n_free", _INT, (1,), self.device)
        self.table, self.pages, self.free, self.n_free, self.page_size = table, pages, free, n_free, int(page_size)

    @classmethod
    def create(cls, n_pages: int, page_size: int, batch: int, max_pages: int, device="cuda") -> "PagePool":
        """A pool whose ``n_pages`` pages are all free."""
        return cls(torch.full((batch, max_pages), -1, dtype=_INT, device=device), torch.zeros(batch, dtype=_INT, device=device),
                   torch.arange(n_pages - 1, -1, -1, dtype=_INT, device=device), torch.full((1,), n_pages, dtype=_INT, device=device), page_size)

    def plan(self, kept, fresh, rows: int, parents=None, mask_words: Optional[int] = None, units: int = 0, chunk: int = 512) -> StepPlan:
        """Plan a step in which request b appends ``fresh[b]`` rows behind its ``kept[b]`` tokens (``mw_paged_plan``).  ``rows``:
        capacity of the row arrays, at least the sum of ``fresh``.  ``parents`` int32 [rows]: trees of at most
        32 * ``mask_words`` nodes (default 8 words); None: chains.  ``units``: pieces that the attention's work is cut into
        (0: requests are not cut), none shorter than ``chunk`` keys.  Tables and stack are updated in place; the plan takes
        effect with ``commit``."""
        dev = self.device
        words = 0 if parents is None else 8 if mask_words is None else int(mask_words)
        if rows < 0 or units < 0 or words < 0:
            _fail("rows, units and mask_words must not be negative")
        k, f = _array(kept, "kept", _INT, (self.batch,), dev), _array(fresh, "fresh", _INT, (self.batch,), dev)
        up = None if parents is None else _array(parents, "parents", _INT, (rows,), dev)
        p = StepPlan(self.batch, rows, words, self.batch + units, self.table.device)
        at_units, at_slots, at_start, at_admitted, at_pages, at_free, at_first, at_positions, at_mask = p._addresses()
        args = _lib.PlanArgs(self.batch, rows, self.page_size, self.free.shape[0], self.max_pages, k, f, up, self.table.data_ptr(),
                             self.table.stride(0), self.pages.data_ptr(), at_pages, self.free.data_ptr(), self.n_free.data_ptr(), at_free, at_start,
                             at_admitted, at_slots, at_positions, at_mask if words else None, words, at_units, at_first, units, chunk)
        _check(_lib.load().mw_paged_plan(C.byref(args), dev, _stream(dev)), "mw_paged_plan")
        return p

    def commit(self, plan: StepPlan) -> None:
        """The pool is now as ``plan`` left it."""
        self.pages.copy_(plan.pages)
        self.n_free.copy_(plan.n_free)


def write(cache: PagedCache, k, v, slots) -> None:
    """Rows ``k``, ``v`` [rows, heads, head_dim] (float16 or bfloat16, any row and head strides) into their ``slots`` (int64
    [rows]; -1 drops a row) of one cache layer (``mw_paged_write``)."""
    dev = cache._one().device
    rows = k.shape[0] if k.dim() else 0
    pk, k_row, k_head = _rows3(k, "k", dev)
    pv, v_row, v_head = _rows3(v, "v", dev)
    if tuple(k.shape[1:]) != (cache.heads, cache.head_dim) or v.shape != k.shape or v.dtype is not k.dtype:
        _fail(f"k and v must be [rows, {cache.heads}, {cache.head_dim}] of one type, got {tuple(k.shape)} and {tuple(v.shape)}")
    at = _array(slots, "slots", torch.int64, (rows,), dev)
    _check(_lib.load().mw_paged_write(C.byref(cache.struct), pk, pv, _FLOATS.get(k.dtype, -1), k_row, k_head, v_row, v_head, at, rows, dev,
                                      _stream(dev)), "mw_paged_write")


def tree_attention(q, cache: PagedCache, table, kept, row_start, units, unit_start, max_nodes: int, mask=None, scale: Optional[float] = None,
                   out=None):
    """Attention of the step's rows over one cache layer (``mw_tree_attention``): ``q`` [rows, n_heads, head_dim] -> the same
    shape.  ``row_start``, ``units``, ``unit_start`` and (trees) ``mask`` are a plan's; ``max_nodes``: the most rows a request has.
    ``scale`` defaults to 1 / sqrt(head_dim)."""
    dev = cache._one().device
    pq, q_row, q_head = _rows3(q, "q", dev)
    rows, heads, dim = q.shape
    if dim != cache.head_dim or q.dtype not in (torch.float16, torch.bfloat16):
        _fail(f"q must be float16 or bfloat16 [rows, heads, {cache.head_dim}], got {q.dtype} {tuple(q.shape)}")
    if table.dim() != 2 or table.dtype is not _INT or table.stride(1) != 1 or table.get_device() != dev:
        _fail(f"table must be int32 [batch, max_pages] with dense rows on cuda:{dev}")
    batch, max_pages = table.shape
    n_units = units.shape[0]
    if out is None:
        out = torch.empty((rows, heads, dim), dtype=q.dtype, device=q.device)
    elif out.shape != q.shape or out.dtype is not q.dtype:
        _fail(f"out must be {q.dtype} {tuple(q.shape)}, got {out.dtype} {tuple(out.shape)}")
    po, o_row, o_head = _rows3(out, "out", dev)
    pm, words = None, 0
    if mask is not None:
        words = mask.shape[1] if mask.dim() == 2 else 0
        pm = _array(mask, "mask", _INT, (rows, None), dev)
    args = _lib.TreeArgs(cache.struct, pq, q_row, q_head, po, o_row, o_head, _FLOATS[q.dtype], heads, rows, batch, int(max_nodes), table.data_ptr(),
                         table.stride(0), max_pages, _array(kept, "kept", _INT, (batch,), dev), _array(row_start, "row_start", _INT, (batch + 1,), dev),
                         _array(units, "units", _INT, (None, 4), dev), _array(unit_start, "unit_start", _INT, (batch + 1,), dev), n_units, pm, words,
                         1.0 / math.sqrt(dim) if scale is None else scale, None, 0)
    lib = _lib.load()
    need = lib.mw_tree_attention_workspace(C.byref(args))
    if need < 0:
        _check(need, "mw_tree_attention")
    if need:
        space = torch.empty(need, dtype=torch.uint8, device=q.device)
        args.workspace, args.workspace_bytes = space.data_ptr(), need
    _check(lib.mw_tree_attention(C.byref(args), dev, _stream(dev)), "mw_tree_attention")
    return out


def accept(logits, tokens, parents, row_start, depth: int, suppress=None):
    """Greedy acceptance of the step's trees (``mw_tree_accept``): ``logits`` [rows, vocab] (float32, float16 or bfloat16, any row
    stride), ``tokens``, ``parents`` int32 [rows] -> best [rows], path [batch, depth], count [batch], out_tokens [batch, depth]."""
    dev = _gpu_of(logits, "logits")
    if logits.dim() != 2 or logits.dtype not in _FLOATS or (logits.stride(1) != 1 and logits.shape[1] > 1):
        _fail(f"logits must be float [rows, vocab] with dense rows, got {logits.dtype} {tuple(logits.shape)}")
    if logits.requires_grad:
        _fail("logits require a gradient, and there is no backward pass")
    rows, vocab = logits.shape
    batch = row_start.shape[0] - 1 if row_start.dim() == 1 else 0
    depth = int(depth)
    if batch < 1 or depth < 1:
        _fail("row_start must have a request at least, and depth be positive")
    tok, up = _array(tokens, "tokens", _INT, (rows,), dev), _array(parents, "parents", _INT, (rows,), dev)
    start = _array(row_start, "row_start", _INT, (batch + 1,), dev)
    sup = None if suppress is None else _array(suppress, "suppress", torch.uint8, (vocab,), dev)
    lib = _lib.load()
    args = _lib.AcceptArgs(logits.data_ptr(), logits.stride(0), _FLOATS[logits.dtype], rows, vocab, batch, depth, sup, tok, up, start)
    need = lib.mw_tree_accept_workspace(C.byref(args))
    if need < 0:
        _check(need, "mw_tree_accept")
    n = batch * depth
    buf = torch.empty(rows + 2 * n + batch + need // 4, dtype=_INT, device=logits.device)
    base = buf.data_ptr()
    args.best, args.path, args.out_tokens, args.count = base, base + 4 * rows, base + 4 * (rows + n), base + 4 * (rows + 2 * n)
    args.workspace, args.workspace_bytes = base + 4 * (rows + 2 * n + batch), need
    _check(lib.mw_tree_accept(C.byref(args), dev, _stream(dev)), "mw_tree_accept")
    return (buf[:rows], buf[rows:rows + n].view(batch, depth), buf[rows + 2 * n:rows + 2 * n + batch],
            buf[rows + n:rows + 2 * n].view(batch, depth))


def compact(cache: PagedCache, table, kept, path, count) -> None:
    """Move the accepted rows (``path`` [batch, depth], ``count`` [batch] of ``accept``) to positions kept, kept + 1, ... in every
    layer of ``cache`` (``mw_paged_compact``)."""
    dev = cache.device
    if table.dim() != 2 or table.dtype is not _INT or table.stride(1) != 1 or table.get_device() != dev:
        _fail(f"table must be int32 [batch, max_pages] with dense rows on cuda:{dev}")
    batch, max_pages = table.shape
    layers, stride = (1, 0) if cache.layers is None else (cache.layers, cache.k.stride(0))
    columns = path.shape[1] if path.dim() == 2 else 0
    _check(_lib.load().mw_paged_compact(C.byref(cache.struct), layers, stride, table.data_ptr(), table.stride(0), max_pages,
                                        _array(kept, "kept", _INT, (batch,), dev), _array(path, "path", _INT, (batch, None), dev), columns,
                                        _array(count, "count", _INT, (batch,), dev), batch, dev, _stream(dev)), "mw_paged_compact")
