"""Grouped-head dot-product attention in 16 bits, for serving (forward only):
attention over packed prompts, a paged key-value cache (16-bit, or quantised to int8 / e4m3
as it is written) and the attention of one new token over it.

    out = gqa_attention(q, k, v, cu_q)                       # whole prompts
    cache = GqaCache(n_layers, n_kv_head, head_dim, max_seqs, max_ctx, n_pages, dtype, store="e4m3")
    cache.reserve(seq, n); cache.write(layer, k, v, seqs, cu)
    out = cache.decode(layer, q, seqs)                       # one new token each

Tensors are torch CUDA tensors, bf16 or fp16, used in place on torch's
current stream; q, k and v may be slices of a fused projection's rows (only
the last dimension has to be contiguous).  Index arrays (``cu``, ``start``,
``slots``) are int32 CUDA tensors, which the host does not read, or host
sequences, which are checked (not while a CUDA graph is captured).  Tensors that want a
gradient are refused where autograd records.  The work runs in the CUDA library
(``wb_gqa_*``, include/wave_b200.h); there is no CPU path.
"""
from __future__ import annotations

import struct

import numpy as np

from . import _lib
from .runtime import Context, default_context

try:  # the package imports without torch; these entry points take torch tensors
    import torch
    _DTYPES = {torch.bfloat16: _lib.WB_BF16, torch.float16: _lib.WB_F16}
    _STORES = {**_DTYPES, torch.int8: _lib.WB_INT8, torch.float8_e4m3fn: _lib.WB_E4M3}
    _raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)
except Exception:  # pragma: no cover
    torch, _DTYPES, _STORES, _raw_stream = None, {}, {}, None

PAGE = 128  # positions per page (WB_KV_PAGE)
_INT32 = np.dtype(np.int32)


# wb_gqa_attn_desc and wb_gqa_cache_desc (include/wave_b200.h) in C's layout
_ATTN = struct.Struct("@6if2q3P6q2PP2qP")
_CACHE = struct.Struct("@7i6P")


def _row(head_dim: int) -> int:
    """Stored columns of a head: head_dim up to whole 16s."""
    return -(-head_dim // 16) * 16


def _elsewhere(a: int, b: int):
    return ValueError(f"tensors on devices {a} and {b} (-1 is the host)")


def _entries(a) -> int:
    return a.shape[0] if isinstance(a, torch.Tensor) and a.dim() == 1 else len(a)


def _index(a, n: int, name: str, device: int):
    """(address, object to keep) of an int32 index array of n entries; None is (0, None)."""
    if a is None:
        return 0, None
    if isinstance(a, torch.Tensor) and (at := a.get_device()) >= 0:
        shape = a.shape
        if a.dtype is not torch.int32 or len(shape) != 1 or not a.is_contiguous():
            raise ValueError(f"{name} must be a contiguous int32 vector")
        if at != device:
            raise _elsewhere(device, at)
        keep, size, ptr = a, shape[0], a.data_ptr()
    else:
        given = np.asarray(a.numpy() if isinstance(a, torch.Tensor) else a)
        kind, size = given.dtype, given.size
        if given.ndim != 1 or (size and kind.kind not in "iu"):
            raise ValueError(f"{name} must be a vector of integers")
        keep = np.ascontiguousarray(given, dtype=np.int32)
        if kind is not _INT32 and keep.astype(kind).tobytes() != given.tobytes():
            raise ValueError(f"{name} must be in int32's range")
        ptr = keep.ctypes.data
    if size != n:
        raise ValueError(f"{name} must have {n} entries, has {size}")
    return ptr, keep


def _rows(x, name: str, dtype=None):
    """Strides of [tokens][heads][head_dim] rows, checked."""
    if not isinstance(x, torch.Tensor) or not x.is_cuda or x.dim() != 3:
        raise ValueError(f"{name} must be a CUDA tensor [tokens][heads][head_dim]")
    t = x.dtype
    if t not in _DTYPES or (dtype is not None and t is not dtype):
        raise ValueError(f"{name} must be bfloat16 or float16, as the others")
    if x.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{name} wants a gradient, which these operators do not give: call them under torch.no_grad()")
    ts, hs, ds = x.stride()
    if ds != 1 and x.shape[2] != 1:
        raise ValueError(f"{name}'s last dimension must be contiguous")
    if not x.shape[2]:
        raise ValueError(f"{name} has a head_dim of 0")
    return ts, hs


def _context(ctx, index: int) -> Context:
    """The context for a device, on torch's current stream there."""
    if ctx is None:
        ctx = default_context(index)
    elif ctx.device != index:
        raise ValueError("the context is on another device")
    stream = torch.cuda.current_stream(index).cuda_stream if _raw_stream is None else _raw_stream(index)
    if ctx.stream != stream:
        ctx.set_stream(stream)
    return ctx


def _out(out, q):
    """Strides of a caller's output, checked."""
    if out.shape != q.shape or out.dtype != q.dtype or out.device != q.device:
        raise ValueError(f"out must be {tuple(q.shape)} {q.dtype} on {q.device}")
    return _rows(out, "out", q.dtype)


def gqa_attention(q, k, v, cu_q, cu_k=None, *, causal: bool = True, scale: float | None = None,
                  return_lse: bool = False, out=None, ctx: Context | None = None):
    """Attention over packed prompts (wb_gqa_attention).

    q [tokens][n_head][head_dim]; k, v [tokens][n_kv_head][head_dim]; sequence
    b's rows are cu[b] .. cu[b+1]-1 (``cu_k`` None: as ``cu_q``).  ``scale``
    None: head_dim ** -0.5.  Returns out like q, and with ``return_lse`` also
    the log sum exp of every query's scores, [n_head][tokens] fp32."""
    q_ts, q_hs = _rows(q, "q")
    dtype, device = q.dtype, q.get_device()
    k_ts, k_hs = _rows(k, "k", dtype)
    v_ts, v_hs = _rows(v, "v", dtype)
    Tq, H, hd = q.shape
    Tk, Hkv, k_hd = shape = k.shape
    if v.shape != shape or k_hd != hd:
        raise ValueError("k and v must be [tokens][n_kv_head][head_dim], head_dim as q's")
    if k.get_device() != device or v.get_device() != device:
        raise _elsewhere(device, k.get_device() if k.get_device() != device else v.get_device())
    n_seq = _entries(cu_q) - 1
    if n_seq < 0:
        raise ValueError("cu_q must have one entry more than there are sequences")
    pq, keep_q = _index(cu_q, n_seq + 1, "cu_q", device)
    pk, keep_k = _index(cu_k, n_seq + 1, "cu_k", device)
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
        o_ts, o_hs = H * hd, hd
    else:
        o_ts, o_hs = _out(out, q)
    lse = q.new_empty((H, Tq), dtype=torch.float32) if return_lse else None
    ctx = _context(ctx, device)
    d = _ATTN.pack(_DTYPES[dtype], H, Hkv, hd, n_seq, bool(causal), hd ** -0.5 if scale is None else scale, Tq, Tk,
                   q.data_ptr(), k.data_ptr(), v.data_ptr(), q_ts, q_hs, k_ts, k_hs, v_ts, v_hs, pq, pk,
                   out.data_ptr(), o_ts, o_hs, 0 if lse is None else lse.data_ptr())
    _lib.call("wb_gqa_attention", ctx.handle, d)
    return (out, lse) if return_lse else out


def _cache_desc(k_pages, v_pages, k_scale, v_scale, table, lens, dtype, head_dim):
    shape, kind, index = k_pages.shape, k_pages.dtype, k_pages.get_device()
    if len(shape) != 4 or v_pages.shape != shape or v_pages.dtype is not kind:
        raise ValueError("k_pages and v_pages must be [n_pages][n_kv_head][128][row]")
    n_pages, Hkv, page, row = shape
    store = _STORES.get(kind)
    if store is None or page != PAGE or row != _row(head_dim):
        raise ValueError(f"pages must hold {PAGE} rows of {_row(head_dim)} bf16, fp16, int8 or float8_e4m3fn values")
    good = _held(k_pages, index) and _held(v_pages, index) and _held(table, index)
    ks = vs = 0
    if store == _lib.WB_INT8 or store == _lib.WB_E4M3:
        scales = (n_pages, Hkv, page)
        for x in (k_scale, v_scale):
            if x is None or x.shape != scales or x.dtype is not torch.float32:
                raise ValueError("an 8-bit cache needs fp32 k_scale and v_scale [n_pages][n_kv_head][128]")
        good = good and _held(k_scale, index) and _held(v_scale, index)
        ks, vs = k_scale.data_ptr(), v_scale.data_ptr()
    if table.dim() != 2 or table.dtype is not torch.int32:
        raise ValueError("table must be int32 [n_slots][max_pages]")
    n_slots, max_pages = table.shape
    pl = 0
    if lens is not None:
        if lens.dtype is not torch.int32 or lens.shape != (n_slots,):
            raise ValueError("lens must be int32 [n_slots]")
        good = good and _held(lens, index)
        pl = lens.data_ptr()
    if not good or index < 0:
        raise ValueError("cache arrays must be contiguous CUDA tensors of one device")
    return _CACHE.pack(_DTYPES[dtype], store, Hkv, head_dim, n_pages, n_slots, max_pages,
                       k_pages.data_ptr(), v_pages.data_ptr(), ks, vs, table.data_ptr(), pl)


def _held(x, index: int) -> bool:
    return x.get_device() == index and x.is_contiguous()


def _n_seq(table, cu, slots, rows=None):
    if cu is not None:
        return _entries(cu) - 1
    if slots is not None:
        return _entries(slots)
    return int(table.shape[0] if rows is None else rows)


def gqa_cache_write(k, v, k_pages, v_pages, table, lens, *, cu=None, start=None, slots=None, k_scale=None,
                    v_scale=None, ctx: Context | None = None) -> None:
    """Write packed rows into a paged cache (wb_gqa_cache_write).

    Sequence i's rows cu[i] .. cu[i+1]-1 of k and v [tokens][n_kv_head]
    [head_dim] become positions start[i], .. of slot slots[i] and set its
    length.  ``cu`` None: one row per sequence; ``start`` None: append;
    ``slots`` None: 0, 1, .."""
    k_ts, k_hs = _rows(k, "k")
    dtype, device = k.dtype, k.get_device()
    v_ts, v_hs = _rows(v, "v", dtype)
    total, Hkv, hd = shape = k.shape
    if v.shape != shape or Hkv != k_pages.shape[1]:
        raise ValueError("k and v must be [tokens][n_kv_head][head_dim]")
    d = _cache_desc(k_pages, v_pages, k_scale, v_scale, table, lens, dtype, hd)
    for x in (v, k_pages):
        if x.get_device() != device:
            raise _elsewhere(device, x.get_device())
    n_seq = _n_seq(table, cu, slots, total)
    pc, keep_c = _index(cu, n_seq + 1, "cu", device)
    ps, keep_s = _index(start, n_seq, "start", device)
    pl, keep_l = _index(slots, n_seq, "slots", device)
    ctx = _context(ctx, device)
    _lib.call("wb_gqa_cache_write", ctx.handle, d, pl, n_seq, pc, total, ps, k.data_ptr(), k_ts, k_hs,
              v.data_ptr(), v_ts, v_hs)


def gqa_cache_read(k_pages, v_pages, table, *, head_dim: int, dtype, cu=None, total: int | None = None, start=None,
                   slots=None, k_scale=None, v_scale=None, ctx: Context | None = None):
    """Read positions back (wb_gqa_cache_read): (k, v), each [total]
    [n_kv_head][head_dim] of ``dtype``, packed as in ``gqa_cache_write``
    (``start`` None: from position 0).  ``total`` may be left out when ``cu``
    is None or on the host."""
    if dtype not in _DTYPES:
        raise ValueError("dtype must be bfloat16 or float16")
    d = _cache_desc(k_pages, v_pages, k_scale, v_scale, table, None, dtype, head_dim)
    device = k_pages.get_device()
    n_seq = _n_seq(table, cu, slots)
    if total is None:
        if cu is not None and isinstance(cu, torch.Tensor) and cu.is_cuda:
            raise ValueError("total must be given when cu is on the device")
        total = n_seq if cu is None else int(cu[-1])
    pc, keep_c = _index(cu, n_seq + 1, "cu", device)
    ps, keep_s = _index(start, n_seq, "start", device)
    pl, keep_l = _index(slots, n_seq, "slots", device)
    k = k_pages.new_empty((total, k_pages.shape[1], head_dim), dtype=dtype)
    v = torch.empty_like(k)
    ctx = _context(ctx, device)
    _lib.call("wb_gqa_cache_read", ctx.handle, d, pl, n_seq, pc, total, ps, k.data_ptr(), v.data_ptr())
    return k, v


def gqa_decode(q, k_pages, v_pages, table, lens, *, slots=None, k_scale=None, v_scale=None,
               scale: float | None = None, return_lse: bool = False, out=None, ctx: Context | None = None):
    """Attention of one new token per sequence over its cached positions
    (wb_gqa_decode): q [n_seq][n_head][head_dim] -> out like q (and lse
    [n_seq][n_head] fp32).  Write the token's own key and value first."""
    q_ss, q_hs = _rows(q, "q")
    device = q.get_device()
    n_seq, H, hd = q.shape
    d = _cache_desc(k_pages, v_pages, k_scale, v_scale, table, lens, q.dtype, hd)
    if k_pages.get_device() != device:
        raise _elsewhere(device, k_pages.get_device())
    pl, keep_l = _index(slots, n_seq, "slots", device)
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    else:
        _out(out, q)
        if not out.is_contiguous():
            raise ValueError("out must be contiguous")
    lse = q.new_empty((n_seq, H), dtype=torch.float32) if return_lse else None
    ctx = _context(ctx, device)
    _lib.call("wb_gqa_decode", ctx.handle, d, pl, n_seq, H, q.data_ptr(), q_ss, q_hs,
              hd ** -0.5 if scale is None else scale, out.data_ptr(), 0 if lse is None else lse.data_ptr())
    return (out, lse) if return_lse else out


class GqaCache:
    """A paged cache of n_layers layers for max_seqs sequences of up to
    max_ctx positions, sharing one pool of n_pages pages of 128 positions
    (every layer holds the pool once; a sequence's page ids are the same in
    all of them).  ``store``: "native" (values of ``dtype``), "int8" or
    "e4m3".  Lengths are per layer: a layer's write advances its own."""

    def __init__(self, n_layers: int, n_kv_head: int, head_dim: int, max_seqs: int, max_ctx: int, n_pages: int,
                 dtype=None, store: str = "native", device: int = 0, ctx: Context | None = None):
        dtype = torch.bfloat16 if dtype is None else dtype
        kinds = {"native": dtype, "int8": torch.int8, "e4m3": torch.float8_e4m3fn}
        if dtype not in _DTYPES or store not in kinds:
            raise ValueError('dtype must be bfloat16 or float16, store "native", "int8" or "e4m3"')
        if min(n_layers, n_kv_head, head_dim, max_seqs, max_ctx, n_pages) < 1 or head_dim > 128:
            raise ValueError("bad cache dimensions (head_dim 1 .. 128)")
        self.ctx, self.dtype, self.head_dim = ctx, dtype, head_dim
        self.max_pages = -(-max_ctx // PAGE)
        dev = torch.device("cuda", device if ctx is None else ctx.device)
        shape = (n_layers, n_pages, n_kv_head, PAGE, _row(head_dim))
        self.k_pages = torch.zeros(shape, dtype=torch.uint8 if store != "native" else dtype, device=dev).view(kinds[store])
        self.v_pages = torch.zeros_like(self.k_pages)
        scale = lambda: torch.ones(shape[:-1], device=dev) if store != "native" else [None] * n_layers  # noqa: E731
        self.k_scale, self.v_scale = scale(), scale()
        self.table = torch.full((max_seqs, self.max_pages), -1, dtype=torch.int32, device=dev)
        self.lens = torch.zeros((n_layers, max_seqs), dtype=torch.int32, device=dev)
        # one layer's arrays: indexing them anew costs more than the rest of a call
        self._layer = [(k, v, self.table, n, {"k_scale": ks, "v_scale": vs, "ctx": ctx}) for k, v, n, ks, vs in
                       zip(self.k_pages, self.v_pages, self.lens, self.k_scale, self.v_scale)]
        self._free = list(range(n_pages - 1, -1, -1))
        self._held = [[] for _ in range(max_seqs)]

    def reserve(self, seq: int, n_positions: int) -> None:
        """Pages so that slot ``seq`` holds ``n_positions`` positions."""
        held, need = self._held[seq], -(-n_positions // PAGE)
        if need > self.max_pages:
            raise ValueError("n_positions exceeds max_ctx")
        more = need - len(held)
        if more <= 0:
            return
        if more > len(self._free):
            raise RuntimeError(f"out of cache pages ({len(self._free)} free, {more} needed)")
        new = [self._free.pop() for _ in range(more)]
        self.table[seq, len(held):need] = torch.tensor(new, dtype=torch.int32, device=self.table.device)
        held += new

    def release(self, seq: int) -> None:
        """Empty slot ``seq`` and return its pages to the pool.  Work already
        queued on the current stream still sees the slot as it was; later
        work on that stream does not."""
        self.table[seq].fill_(-1)
        self.lens[:, seq].fill_(0)
        self._free += reversed(self._held[seq])
        self._held[seq] = []

    def free_pages(self) -> int:
        return len(self._free)

    def write(self, layer: int, k, v, slots=None, cu=None, start=None) -> None:
        """gqa_cache_write into one layer."""
        k_pages, v_pages, table, lens, more = self._layer[layer]
        gqa_cache_write(k, v, k_pages, v_pages, table, lens, cu=cu, start=start, slots=slots, **more)

    def read(self, layer: int, slots=None, cu=None, total: int | None = None, start=None):
        """gqa_cache_read from one layer, in the cache's dtype."""
        k_pages, v_pages, table, _, more = self._layer[layer]
        return gqa_cache_read(k_pages, v_pages, table, head_dim=self.head_dim, dtype=self.dtype, cu=cu, total=total,
                              start=start, slots=slots, **more)

    def decode(self, layer: int, q, slots=None, *, scale: float | None = None, return_lse: bool = False, out=None):
        """gqa_decode over one layer."""
        k_pages, v_pages, table, lens, more = self._layer[layer]
        return gqa_decode(q, k_pages, v_pages, table, lens, slots=slots, scale=scale, return_lse=return_lse, out=out,
                          **more)
