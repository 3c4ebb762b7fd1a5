"""Batched serving over a paged cache (include/xalm_cuda.h, xalm_cuda_paged_*): torch tensors on a GPU in and out.

    cache = PagedCache(k, v, means)                       # pools (pages, page_size, kv_heads, dim), any nesting of slots and heads
    batch = Batch(starts, lens, table)                    # int32 tensors that a captured graph may rewrite in place
    q = append(cache, batch, k_rows, v_rows, q=q_rows, freq=freq)
    out = attend(cache, batch, q, scale)                  # every page, or
    pages = select(cache, batch, q, top=32)               # the pages worth reading
    out = attend_selected(cache, batch, q, pages, scale)

Calls enqueue kernels on the current stream of the cache's device.  What the host can check is refused with XalmError; what only the device sees
(a table that names no page of the pool, lengths beyond the table) is kept in `cache.status` and raised by cache.check().
"""
from __future__ import annotations

import ctypes as C

import torch

from . import capi
from . import types as T

_TYPES = {torch.float32: T.F32.id, torch.float16: T.F16.id, torch.bfloat16: T.BF16.id}
_INVALID, _UNSUPPORTED = 1, 2
_stream = torch._C._cuda_getCurrentRawStream  # what torch.cuda.current_stream(device).cuda_stream says, in a twentieth of its 2 us


class _Cache(C.Structure):
    _fields_ = [(n, C.c_int) for n in ("type", "device", "pages", "page_size", "kv_heads", "dim", "vdim")] + [("k", C.c_void_p), ("v", C.c_void_p)] + \
               [(n, C.c_longlong) for n in ("k_page", "k_slot", "k_head", "v_page", "v_slot", "v_head")] + [("means", C.c_void_p), ("status", C.c_void_p)]


class _Batch(C.Structure):
    _fields_ = [(n, C.c_int) for n in ("rows", "seqs", "max_pages", "groups")] + [(n, C.c_void_p) for n in ("starts", "lens", "table")] + \
               [("table_row", C.c_longlong), ("group_bounds", C.c_void_p), ("group_shared", C.c_void_p)]


def _refuse(why, status=_INVALID):
    raise capi.XalmError(status, why)


def _type(t):
    if t.dtype not in _TYPES:
        _refuse(f"paged cache: {t.dtype} (float32, float16 and bfloat16)", _UNSUPPORTED)
    return _TYPES[t.dtype]


class PagedCache:
    """Pools of keys (pages, page_size, kv_heads, dim) and values (.., vdim), both of the caller; the last dimension's entries are neighbours.  means
    (pages, kv_heads, dim), contiguous, or None."""

    def __init__(self, k, v, means=None):
        if k.dim() != 4 or v.dim() != 4 or k.shape[:3] != v.shape[:3] or k.dtype != v.dtype or k.device != v.device:
            _refuse(f"paged cache: keys {tuple(k.shape)} {k.dtype} and values {tuple(v.shape)} {v.dtype}")
        if k.stride(3) != 1 or v.stride(3) != 1:
            _refuse("paged cache: the entries of a head are neighbours")
        if means is not None and (means.shape != (k.shape[0], k.shape[2], k.shape[3]) or means.dtype != k.dtype or means.device != k.device or not means.is_contiguous()):
            _refuse(f"paged cache: mean keys {tuple(means.shape)} {means.dtype}")
        self.k, self.v, self.means, self.device, self.index, self.dtype = k, v, means, k.device, k.device.index, k.dtype
        self.needs = {}  # bytes of workspace by the sizes of a call
        self.kv_heads, self.dim, self.vdim = k.shape[2], k.shape[3], v.shape[3]
        if k.device.type != "cuda":
            _refuse("paged cache: the pools lie on no GPU")
        self.status = torch.zeros(1, dtype=torch.int32, device=k.device)

        def strides(t):  # a dimension of one entry has no stride of its own
            page, slot, head, _ = t.stride()
            return page if t.shape[0] > 1 else 1 << 36, slot, head if t.shape[2] > 1 else t.shape[3]

        self.c = _Cache(_type(k), k.device.index, k.shape[0], k.shape[1], k.shape[2], k.shape[3], v.shape[3], k.data_ptr(), v.data_ptr(), *strides(k), *strides(v),
                        0 if means is None else means.data_ptr(), self.status.data_ptr())
        self.p = C.addressof(self.c)

    def check(self):
        """Waits for the device, all its streams, and raises what its kernels have reported since the last check.  Not while a graph is captured."""
        torch.cuda.synchronize(self.device)
        taken = torch.empty_like(self.status)
        capi.check(capi.lib().xalm_cuda_paged_status(self.p, taken.data_ptr(), _stream(self.index)))
        bits = int(taken.item())
        if bits:
            _refuse("paged cache: " + " and ".join(t for b, t in ((1, "a table names a page outside the pool"), (2, "starts, lens and table do not fit"), (4, "a kernel gave up a wait for its copies or products")) if bits & b))


class Batch:
    """starts (seqs + 1), lens (seqs), table (seqs, max_pages): int32, on the cache's device.  groups (n + 1) and shared (n): sequences groups[i] .. groups[i + 1] - 1
    have their first shared[i] tokens' pages in common."""

    def __init__(self, starts, lens, table, groups=None, shared=None):
        tensors = [starts, lens, table] + ([] if groups is None else [groups, shared])
        if (groups is None) != (shared is None):
            _refuse("paged batch: groups and shared come together")
        if any(t.dtype != torch.int32 or t.device != starts.device for t in tensors):
            _refuse("paged batch: int32 tensors of one device")
        if table.dim() != 2 or starts.shape != (table.shape[0] + 1,) or lens.shape != (table.shape[0],) or (groups is not None and (groups.dim() != 1 or groups.shape[0] != shared.numel() + 1 or shared.dim() != 1)):
            _refuse(f"paged batch: starts {tuple(starts.shape)}, lens {tuple(lens.shape)}, table {tuple(table.shape)}")
        if any(t.numel() > 1 and t.stride(-1) != 1 for t in tensors):
            _refuse("paged batch: entries are neighbours")
        self.tensors, self.device, self.seqs = tensors, starts.device, table.shape[0]
        row = table.stride(0) if table.shape[0] > 1 else table.shape[1]
        self.c = _Batch(0, table.shape[0], table.shape[1], 0 if groups is None else shared.shape[0], starts.data_ptr(), lens.data_ptr(), table.data_ptr(), row,
                        0 if groups is None else groups.data_ptr(), 0 if groups is None else shared.data_ptr())
        self.p = C.addressof(self.c)
        self.sized = {}  # the same with a call's number of rows, which calls in other threads do not change

    def of(self, rows):
        c = self.sized.get(rows)
        if c is None:
            if len(self.sized) > 1000:
                self.sized.clear()
            c = _Batch.from_buffer_copy(self.c)
            c.rows = rows
            c = self.sized[rows] = (C.addressof(c), c)
        return c


def _rows(t, what, n, heads, dim, dtype, device):
    """Row stride of (n, heads, dim) rows whose heads are dense."""
    if t.shape != (n, heads, dim):
        _refuse(f"paged cache: {what} {tuple(t.shape)}, not ({n}, {heads}, {dim})")
    if t.dtype is not dtype or t.device != device:
        _refuse(f"paged cache: {what} is {t.dtype} on {t.device}")
    row, head, entry = t.stride()
    if entry != 1 or (head != dim and heads > 1):
        _refuse(f"paged cache: the heads of {what} are dense")
    return row if n > 1 else heads * dim


def _start(cache, batch, rows):
    if batch.device != cache.device:
        _refuse(f"paged cache: a batch on {batch.device}, a cache on {cache.device}")
    return batch.of(rows), _stream(cache.index)


def _heads(q):
    if q.dim() != 3:
        _refuse(f"paged cache: q {tuple(q.shape)}, not (rows, heads, dim)")
    return q.shape[1]


def _beside(q, n, heads, dim, cache):
    """(n, heads, dim) of the cache's type, in the quickest way: torch.empty takes 1 us longer, Tensor.new_empty half of one."""
    if dim == cache.dim and q.dtype is cache.dtype and q.is_contiguous():
        return torch.empty_like(q)
    return q.new_empty((n, heads, dim), dtype=cache.dtype)


def append(cache, batch, k, v, q=None, freq=None, mag=1.0, neighbours=False, q_out=None):
    """k (rows, kv_heads, dim) and v (rows, kv_heads, vdim) into the pages of their sequences; returns the turned queries in the cache's type (None without q).  freq
    (n): the first 2 n entries of every head are turned."""
    n, dev, dt = k.shape[0], cache.device, k.dtype
    (bp, held), stream = _start(cache, batch, n)
    kr, vr = _rows(k, "k", n, cache.kv_heads, cache.dim, dt, dev), _rows(v, "v", n, cache.kv_heads, cache.vdim, dt, dev)
    qr = qor = heads = qp = qop = fp = rot = 0
    if q is not None:
        heads = _heads(q)
        qr = _rows(q, "q", n, heads, cache.dim, dt, dev)
        if q_out is None:
            q_out = _beside(q, n, heads, cache.dim, cache)
            qor = heads * cache.dim
        else:
            qor = _rows(q_out, "q_out", n, heads, cache.dim, cache.dtype, dev)
        qp, qop = q.data_ptr(), q_out.data_ptr()
    elif q_out is not None:
        _refuse("paged append: q_out without q")
    if freq is not None:
        if freq.dtype is not torch.float32 or freq.dim() != 1 or not freq.is_contiguous() or freq.device != dev:
            _refuse(f"paged append: freq {tuple(freq.shape)} {freq.dtype} on {freq.device}")
        fp, rot = freq.data_ptr(), freq.shape[0]
    capi.check(capi.lib().xalm_cuda_paged_append(cache.p, bp, k.data_ptr(), kr, v.data_ptr(), vr, qp, qr, heads, _type(k), qop, qor, fp, rot, mag, neighbours, stream))
    return q_out


def _attend(cache, batch, q, lists, scale, out, want_lse):
    heads, n, dev = _heads(q), q.shape[0], cache.device
    (bp, held), stream = _start(cache, batch, n)
    qr = _rows(q, "q", n, heads, cache.dim, cache.dtype, dev)
    if out is None:
        out = _beside(q, n, heads, cache.vdim, cache)
        outr = heads * cache.vdim
    else:
        outr = _rows(out, "out", n, heads, cache.vdim, cache.dtype, dev)
    lse = q.new_empty((n, heads), dtype=torch.float32) if want_lse else None
    s, L = 0 if lists is None else lists.shape[2], capi.lib()
    sizes = n, heads, s, batch.c.seqs, batch.c.groups
    need = cache.needs.get(sizes)
    if need is None:
        b = C.c_size_t(0)
        capi.check(L.xalm_cuda_paged_workspace(cache.p, bp, heads, s, C.byref(b)))
        if len(cache.needs) > 1000:
            cache.needs.clear()
        need = cache.needs[sizes] = b.value
    work = q.new_empty(need, dtype=torch.uint8)  # the current stream's, or the graph's that is being captured
    lp = None if lse is None else lse.data_ptr()
    if lists is None:
        capi.check(L.xalm_cuda_paged_attend(cache.p, bp, q.data_ptr(), qr, heads, scale, out.data_ptr(), outr, lp, work.data_ptr(), need, stream))
    else:
        capi.check(L.xalm_cuda_paged_attend_selected(cache.p, bp, q.data_ptr(), qr, heads, lists.data_ptr(), s, scale, out.data_ptr(), outr, lp, work.data_ptr(), need, stream))
    return (out, lse) if want_lse else out


def attend(cache, batch, q, scale, out=None, want_lse=False):
    """q (rows, heads, dim) of the cache's type; returns (rows, heads, vdim), and with want_lse the logarithms of the denominators (rows, heads) too.  Rows outside every
    sequence are left as they were."""
    return _attend(cache, batch, q, None, scale, out, want_lse)


def select(cache, batch, q, top, first=1, recent=1, out=None):
    """The `top` pages that each row and kv head reads: (rows, kv_heads, top) int32, places in the sequence, ascending, -1 behind; rows outside every sequence are left as they were."""
    heads, n, dev = _heads(q), q.shape[0], cache.device
    (bp, held), stream = _start(cache, batch, n)
    qr = _rows(q, "q", n, heads, cache.dim, cache.dtype, dev)
    if out is None:
        out = q.new_empty((n, cache.kv_heads, max(top, 0)), dtype=torch.int32)
    elif out.shape != (n, cache.kv_heads, top) or out.dtype != torch.int32 or not out.is_contiguous() or out.device != dev:
        _refuse(f"paged select: out {tuple(out.shape)} {out.dtype}")
    capi.check(capi.lib().xalm_cuda_paged_select(cache.p, bp, q.data_ptr(), qr, heads, top, first, recent, out.data_ptr(), stream))
    return out


def attend_selected(cache, batch, q, pages, scale, out=None, want_lse=False):
    """attend over the pages of `pages` (rows, kv_heads, n) only, as select gives them or in any other order."""
    if pages.dim() != 3 or pages.shape[:2] != (q.shape[0], cache.kv_heads) or pages.dtype != torch.int32 or not pages.is_contiguous() or pages.device != cache.device:
        _refuse(f"paged attention: lists {tuple(pages.shape)} {pages.dtype}")
    return _attend(cache, batch, q, pages, scale, out, want_lse)
