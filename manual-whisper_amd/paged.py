"""Drafted tokens over a K/V cache in pages: the operators of one step of drafted decoding on torch tensors.

    pool = PagePool.create(n_pages, page_size, batch, max_pages)       # tables and the stack of free pages
    cache = PagedCache.empty(layers, n_pages, heads, page_size, head_dim)
    plan = pool.plan(kept, fresh, rows, parents, units=256)            # pages, slots, positions, masks, work units
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
is kept between calls.  There is no derivative, backward or forward: a tensor that requires a gradient is taken under
``torch.no_grad()`` only, one with a tangent never.  A bad argument raises ``EngineError``.
"""
from __future__ import annotations

import ctypes as C
import math
import struct
from typing import Optional

import torch
from torch.autograd import forward_ad

from . import _lib
from .engine import EngineError

_FLOATS = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
_HALVES = (torch.float16, torch.bfloat16)
_CODES = (torch.uint8, torch.float8_e4m3fn)
_E4M3 = 3
_INT = torch.int32


# A call here is a launch of a few microseconds, so the argument structs of include/mwhip.h are packed with `struct` (native
# alignment, like the compiler's) rather than filled in field by field.
def _codec(fields):
    kinds = {C.c_void_p: "P", C.c_int64: "q", C.c_int32: "i", C.c_float: "f"}
    return "".join(_codec(t._fields_) if hasattr(t, "_fields_") else kinds[t] for _, t in fields)


_CACHE = struct.Struct("@" + _codec(_lib.PagedCache._fields_) + "0P")
_PLAN = struct.Struct("@" + _codec(_lib.PlanArgs._fields_) + "0P")
_ACCEPT = struct.Struct("@" + _codec(_lib.AcceptArgs._fields_) + "0P")
_TREE = struct.Struct("@" + _codec(_lib.TreeArgs._fields_) + "0P")
_calls = None


class _Calls:
    """The entry points with their struct arguments as bytes."""

    def __init__(self):
        lib = _lib.load()
        by, i32, i64, vp = C.c_char_p, C.c_int32, C.c_int64, C.c_void_p

        def fn(name, res, *args):
            return C.CFUNCTYPE(res, *args)((name, lib))

        self.plan = fn("mw_paged_plan", i32, by, i32, vp)
        self.write = fn("mw_paged_write", i32, by, vp, vp, i32, i64, i64, i64, i64, vp, i64, i32, vp)
        self.tree_space = fn("mw_tree_attention_workspace", i64, by)
        self.tree = fn("mw_tree_attention", i32, by, i32, vp)
        self.accept_space = fn("mw_tree_accept_workspace", i64, by)
        self.accept = fn("mw_tree_accept", i32, by, i32, vp)
        self.compact = fn("mw_paged_compact", i32, by, i32, i64, vp, i64, i32, vp, vp, i32, vp, i32, i32, vp)


def _c() -> _Calls:
    global _calls
    if _calls is None:
        _calls = _Calls()
    return _calls


def _fail(what: str):
    raise EngineError(what)


def _failed(rc: int, what: str):
    raise EngineError(f"{what} failed ({rc}): {_lib.load().mw_last_error(None).decode()}")


_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda device: torch.cuda.current_stream(device).cuda_stream)


def _array(t, name: str, dtype, shape, device: int) -> int:
    """Address of a contiguous tensor of the expected type, shape and GPU."""
    if t.dtype is dtype and t.shape == shape and t.get_device() == device and t.is_contiguous():
        return t.data_ptr()
    _fail(f"{name} must be a contiguous {dtype} tensor of shape {tuple(shape)} on cuda:{device}, got {t.dtype} {tuple(t.shape)} "
          f"strides {t.stride()} on {t.device}")


def _gpu_of(t, name: str) -> int:
    if not t.is_cuda:
        _fail(f"{name} must be on a GPU, got {t.device}")
    return t.get_device()


def _table(t, device: int):
    """(address, batch, columns, row stride) of a block table."""
    if t.dtype is not _INT or t.dim() != 2 or t.get_device() != device:
        _fail(f"table must be int32 [batch, max_pages] on cuda:{device}, got {t.dtype} {tuple(t.shape)} on {t.device}")
    stride, inner = t.stride()
    batch, columns = t.shape
    if (inner != 1 and columns > 1) or (stride < columns and batch > 1):
        _fail(f"table must have dense rows of its own, got strides {t.stride()}")
    return t.data_ptr(), batch, columns, stride if batch > 1 else columns        # (the stride of a dimension of one may be anything)


def _no_gradient(t, name: str) -> None:
    """Refuse a tensor that would have to pass a gradient on: there is no backward pass, and none forward either."""
    if t.requires_grad and torch.is_grad_enabled():
        _fail(f"{name} requires a gradient, and there is no backward pass (torch.no_grad() for its values)")
    if forward_ad._current_level >= 0 and forward_ad.unpack_dual(t).tangent is not None:
        _fail(f"{name} has a tangent, and there is no forward-mode derivative")


def _rows3(t, name: str, device: int):
    """(address, row stride, head stride) of a [rows, heads, head_dim] tensor whose last dimension is dense."""
    if t.dim() != 3 or t.get_device() != device:
        _fail(f"{name} must be [rows, heads, head_dim] on cuda:{device}, got {tuple(t.shape)} on {t.device}")
    _no_gradient(t, name)
    row, head, inner = t.stride()
    if inner != 1:
        _fail(f"{name} must have dense rows, got strides {t.stride()}")
    rows, heads, dim = t.shape
    return t.data_ptr(), row if rows > 1 else 0, head if heads > 1 else dim


def _tight(shape, strides):
    return tuple(shape[-1] if n == 1 else s for n, s in zip(shape[:-1], strides)) + strides[-1:]


class PagedCache:
    """K/V in pages: ``k``, ``v`` [layers, pages, heads, page_size, head_dim] (or without the layers: one layer) of float16 or
    bfloat16, or e4m3 codes (uint8 / float8_e4m3fn) with the row scales ``k_scale``, ``v_scale`` (float32, contiguous, the
    shape without head_dim).  The order of pages, heads and tokens in memory is free (transposed views are fine); rows are
    dense and start at multiples of 16 bytes.  ``page_size``: a power of two in 16..4096; ``head_dim``: 64 or 128."""

    def __init__(self, k, v, k_scale=None, v_scale=None):
        shape, strides, dtype = k.shape, k.stride(), k.dtype
        if 1 in shape[:-2] and shape == v.shape:           # the stride of a dimension of one may be anything: the next one's, then
            strides, other = _tight(shape, strides), _tight(shape, v.stride())
        else:
            other = v.stride()
        if len(shape) not in (4, 5) or shape != v.shape or dtype is not v.dtype or strides != other:
            _fail(f"k and v must be [(layers,) pages, heads, page_size, head_dim] of one type and layout, got {tuple(shape)} {dtype} "
                  f"and {tuple(v.shape)} {v.dtype}")
        self.device = device = _gpu_of(k, "k")
        codes = dtype in _CODES
        if not codes and dtype not in _HALVES:
            _fail(f"a cache holds float16, bfloat16 or e4m3 codes, got {dtype}")
        if strides[-1] != 1 or v.get_device() != device:
            _fail("rows of the cache must be dense, and k and v on one GPU")
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self.layers = shape[0] if len(shape) == 5 else None
        self.n_pages, self.heads, self.page_size, self.head_dim = shape[-4:]
        ks = vs = 0
        if codes:
            if k_scale is None or v_scale is None:
                _fail("an e4m3 cache needs its row scales")
            ks = _array(k_scale, "k_scale", torch.float32, shape[:-1], device)
            vs = _array(v_scale, "v_scale", torch.float32, shape[:-1], device)
        elif k_scale is not None or v_scale is not None:
            _fail("row scales belong to an e4m3 cache")
        self.dtype = _E4M3 if codes else _FLOATS[dtype]
        self._fields = (k.data_ptr(), v.data_ptr(), ks, vs, *strides[-4:-1], self.n_pages, self.page_size, self.heads, self.head_dim, self.dtype)
        self._bytes = _CACHE.pack(*self._fields)

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

    def __init__(self, batch: int, rows: int, words: int, n_units: int, device):
        sizes = (4 * n_units, 2 * rows, batch + 1, batch, batch, 1, batch + 1, rows, rows * words)
        buf = torch.empty(4 * n_units + 3 * rows + 4 * batch + 3 + rows * words, dtype=_INT, device=device)
        units, slots, self.row_start, self.admitted, self.pages, self.n_free, self.unit_start, self.positions, mask = buf.split_with_sizes(sizes)
        self.units, self.slots = units.view(n_units, 4), slots.view(torch.int64)
        self.mask = mask.view(rows, words) if words else None
        at_units = buf.data_ptr()
        at_slots = at_units + 16 * n_units
        at_start = at_slots + 8 * rows
        at_admitted = at_start + 4 * (batch + 1)
        at_pages = at_admitted + 4 * batch
        at_free = at_pages + 4 * batch
        at_first = at_free + 4
        at_positions = at_first + 4 * (batch + 1)
        self._at = (at_free, at_start, at_admitted, at_slots, at_positions, at_positions + 4 * rows if words else 0, words, at_units, at_first)
        self._at_pages = at_pages


class PagePool:
    """Tables [batch, max_pages], pages held per request [batch] and the stack of free pages [n_pages] with its height [1]."""

    def __init__(self, table, pages, free, n_free, page_size: int):
        self.device = device = _gpu_of(table, "table")
        _, self.batch, self.max_pages, _ = _table(table, device)
        _array(pages, "pages", _INT, (self.batch,), device)
        _array(free, "free", _INT, (free.numel(),), device)
        _array(n_free, "n_free", _INT, (1,), device)
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
        (0: requests are not cut), none shorter than ``chunk`` keys.  Long caches need the cut, or few requests leave most of the
        GPU idle: about 2048 pieces over the cache's heads (``max(16, 2048 // heads)``), ``chunk`` at least 512 and at least 4
        times the query columns of a K/V head (rows of a request times query heads per K/V head); 0 where no request is
        longer than some 512 keys.  Tables and stack are updated in place; the plan takes effect with ``commit``."""
        dev, batch = self.device, self.batch
        words = 0 if parents is None else 8 if mask_words is None else int(mask_words)
        if not (0 <= rows < 1 << 30 and 0 <= units <= 1 << 16 and 1 <= chunk < 1 << 31 and 0 <= words <= 8):
            _fail(f"rows must be in 0..2^30 - 1, units in 0..65536, chunk positive and mask_words at most 8, got {rows}, {units}, {chunk}, {words}")
        k, f = _array(kept, "kept", _INT, (batch,), dev), _array(fresh, "fresh", _INT, (batch,), dev)
        up = 0 if parents is None else _array(parents, "parents", _INT, (rows,), dev)
        p = StepPlan(batch, rows, words, batch + units, self.table.device)
        table, _, columns, stride = _table(self.table, dev)
        args = _PLAN.pack(batch, rows, self.page_size, self.free.shape[0], columns, k, f, up, table, stride, self.pages.data_ptr(), p._at_pages,
                          self.free.data_ptr(), self.n_free.data_ptr(), *p._at, units, chunk)
        rc = _c().plan(args, dev, _raw_stream(dev))
        if rc:
            _failed(rc, "mw_paged_plan")
        return p

    def commit(self, plan: StepPlan) -> None:
        """The pool is now as ``plan`` left it."""
        self.pages.copy_(plan.pages)
        self.n_free.copy_(plan.n_free)


def write(cache: PagedCache, k, v, slots) -> None:
    """Rows ``k``, ``v`` [rows, heads, head_dim] (float16 or bfloat16, any row and head strides) into their ``slots`` (int64
    [rows], all different; -1 drops a row) of one cache layer (``mw_paged_write``)."""
    dev = cache._one().device
    pk, k_row, k_head = _rows3(k, "k", dev)
    pv, v_row, v_head = _rows3(v, "v", dev)
    shape = k.shape
    rows = shape[0]
    if shape != (rows, cache.heads, cache.head_dim) or v.shape != shape or v.dtype is not k.dtype:
        _fail(f"k and v must be [rows, {cache.heads}, {cache.head_dim}] of one type, got {tuple(k.shape)} and {tuple(v.shape)}")
    rc = _c().write(cache._bytes, pk, pv, _FLOATS.get(k.dtype, -1), k_row, k_head, v_row, v_head,
                    _array(slots, "slots", torch.int64, (rows,), dev), rows, dev, _raw_stream(dev))
    if rc:
        _failed(rc, "mw_paged_write")


def tree_attention(q, cache: PagedCache, table, kept, row_start, units, unit_start, max_nodes: int, mask=None, scale: Optional[float] = None,
                   out=None):
    """Attention of the step's rows over one cache layer (``mw_tree_attention``): ``q`` [rows, n_heads, head_dim] -> the same
    shape.  ``row_start``, ``units``, ``unit_start`` and (trees) ``mask`` are a plan's; ``max_nodes``: the most rows a request has.
    ``scale`` defaults to 1 / sqrt(head_dim).  Where requests are cut, the workspace grows with the units times ``max_nodes``: prompts
    are better attended to in a call of their own than among single rows.  Rows behind the last request are left as they are in
    ``out`` (undefined without one)."""
    dev = cache._one().device
    pq, q_row, q_head = _rows3(q, "q", dev)
    rows, heads, dim = q.shape
    if dim != cache.head_dim or q.dtype not in _HALVES:
        _fail(f"q must be float16 or bfloat16 [rows, heads, {cache.head_dim}], got {q.dtype} {tuple(q.shape)}")
    if not 0 <= max_nodes <= 1 << 20:
        _fail(f"max_nodes must be in 0..2^20, got {max_nodes}")
    pt, batch, columns, t_stride = _table(table, dev)
    n_units = units.shape[0]
    if out is None:
        out = q.new_empty(rows, heads, dim)
        po, o_row, o_head = out.data_ptr(), heads * dim, dim
    else:
        if out.shape != q.shape or out.dtype is not q.dtype:
            _fail(f"out must be {q.dtype} {tuple(q.shape)}, got {out.dtype} {tuple(out.shape)}")
        po, o_row, o_head = _rows3(out, "out", dev)
    pm = words = 0
    if mask is not None:
        words = mask.shape[1] if mask.dim() == 2 else 0
        pm = _array(mask, "mask", _INT, (rows, words), dev)
    fields = cache._fields + (pq, q_row, q_head, po, o_row, o_head, _FLOATS[q.dtype], heads, rows, batch, int(max_nodes), pt, t_stride, columns,
                              _array(kept, "kept", _INT, (batch,), dev), _array(row_start, "row_start", _INT, (batch + 1,), dev),
                              _array(units, "units", _INT, (n_units, 4), dev), _array(unit_start, "unit_start", _INT, (batch + 1,), dev), n_units,
                              pm, words, 1.0 / math.sqrt(dim) if scale is None else scale)
    c = _c()
    args = _TREE.pack(*fields, 0, 0)
    if n_units != batch:                                     # requests may be cut: their pieces' results meet in a workspace
        need = c.tree_space(args)
        if need < 0:
            _failed(need, "mw_tree_attention")
        if need:
            space = torch.empty(need, dtype=torch.uint8, device=q.device)
            args = _TREE.pack(*fields, space.data_ptr(), need)
    rc = c.tree(args, dev, _raw_stream(dev))
    if rc:
        _failed(rc, "mw_tree_attention")
    return out


def accept(logits, tokens, parents, row_start, depth: int, suppress=None):
    """Greedy acceptance of the step's trees (``mw_tree_accept``): ``logits`` [rows, vocab] (float32, float16 or bfloat16, any row
    stride), ``tokens``, ``parents`` int32 [rows] -> best [rows] (undefined behind the last request), path [batch, depth], count
    [batch], out_tokens [batch, depth]."""
    dev = _gpu_of(logits, "logits")
    dtype = _FLOATS.get(logits.dtype)
    if logits.dim() != 2 or dtype is None:
        _fail(f"logits must be float [rows, vocab], got {logits.dtype} {tuple(logits.shape)}")
    _no_gradient(logits, "logits")
    rows, vocab = logits.shape
    stride, inner = logits.stride()
    if inner != 1 and vocab > 1:
        _fail(f"logits must have dense rows, got strides {logits.stride()}")
    batch = row_start.shape[0] - 1 if row_start.dim() == 1 else 0
    depth = int(depth)
    if batch < 1 or not 1 <= depth <= 1024:
        _fail("row_start must have a request at least, and depth be in 1..1024")
    head = (logits.data_ptr(), stride, dtype, rows, vocab, batch, depth,
            0 if suppress is None else _array(suppress, "suppress", torch.uint8, (vocab,), dev), _array(tokens, "tokens", _INT, (rows,), dev),
            _array(parents, "parents", _INT, (rows,), dev), _array(row_start, "row_start", _INT, (batch + 1,), dev))
    c = _c()
    need = c.accept_space(_ACCEPT.pack(*head, 0, 0, 0, 0, 0, 0))
    if need < 0:
        _failed(need, "mw_tree_accept")
    n = batch * depth
    sizes = (rows, n, batch, n, need // 4)
    buf = torch.empty(sum(sizes), dtype=_INT, device=logits.device)
    base = buf.data_ptr()
    at_path, at_count = base + 4 * rows, base + 4 * (rows + n)
    at_tokens = at_count + 4 * batch
    rc = c.accept(_ACCEPT.pack(*head, base, at_path, at_count, at_tokens, at_tokens + 4 * n, need), dev, _raw_stream(dev))
    if rc:
        _failed(rc, "mw_tree_accept")
    best, path, count, out, _ = buf.split_with_sizes(sizes)
    return best, path.view(batch, depth), count, out.view(batch, depth)


def compact(cache: PagedCache, table, kept, path, count) -> None:
    """Move the accepted rows (``path`` [batch, depth], ``count`` [batch] of ``accept``) to positions kept, kept + 1, ... in every
    layer of ``cache`` (``mw_paged_compact``)."""
    dev = cache.device
    pt, batch, columns, t_stride = _table(table, dev)
    layers, stride = (1, 0) if cache.layers is None else (cache.layers, cache.k.stride(0))
    depth = path.shape[1] if path.dim() == 2 else 0
    rc = _c().compact(cache._bytes, layers, stride, pt, t_stride, columns, _array(kept, "kept", _INT, (batch,), dev),
                      _array(path, "path", _INT, (batch, depth), dev), depth, _array(count, "count", _INT, (batch,), dev), batch, dev, _raw_stream(dev))
    if rc:
        _failed(rc, "mw_paged_compact")
