"""The paged key-value cache: ``append`` rows of new tokens, ``decode`` one new token per
sequence, ``evict`` the keys that attention has used least.

``core.decode`` runs the thresholded rules over one contiguous cache; here a batch of sequences
of any lengths shares a pool of fixed-size pages.  As everywhere in this package the cache holds
RAW keys: ``decode`` rotates them where it reads them, so one cache serves every geometry
(positions interpolated, YaRN, Dual Chunk Attention), and evicted caches are read at dense ranks
(slot = position), like the sets of the PQ-Union rule.

Every call launches on torch's current stream of the cache's device and reads the lengths on the
device: nothing synchronises, and calls can be captured into CUDA graphs.  The one exception is a
geometry whose ``inv_freq`` lies elsewhere: ``decode`` then copies it on every call, which waits
for the copy, and refuses to be captured.
"""
from __future__ import annotations

import ctypes
import math

import torch

from . import _lib as L
from .core import Geometry, dtype_code


def _on(t, dev, dtype, shape, name):
    """t is a tensor of this device, type and shape (None entries: any) with a dense last dim."""
    if isinstance(t, torch.Tensor) and t.dtype is dtype and t.device == dev:
        s = t.shape
        if len(s) == len(shape):
            for m, n in zip(s, shape):
                if n is not None and m != n:
                    break
            else:
                if not s or s[-1] <= 1 or t.stride(-1) == 1:
                    return
    if not isinstance(t, torch.Tensor) or t.device != dev:
        raise ValueError(f"{name} must be a tensor on {dev}")
    if t.dtype != dtype:
        raise TypeError(f"{name} must be {dtype}, got {t.dtype}")
    if t.dim() != len(shape) or any(n is not None and m != n for m, n in zip(t.shape, shape)):
        raise ValueError(f"{name} has shape {tuple(t.shape)}, expected {tuple(shape)}")
    raise ValueError(f"the last dimension of {name} must be contiguous")


def _run(cache, entry, name, *args):
    """Call a library entry with the cache, on the current stream of the cache's device."""
    dev = cache._index
    if _device() == dev:
        rc = entry(cache._ref, *args, _raw_stream(dev))
    else:
        with torch.cuda.device(dev):
            rc = entry(cache._ref, *args, _raw_stream(dev))
    if rc:
        L.check(rc, name)


# (a torch without CUDA has neither; no cache exists there that could call them)
_device = getattr(torch._C, "_cuda_getDevice", None)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _size(cache, key, entry, name, ref):
    """Bytes of scratch that a call needs (by the shapes alone, so asked for once).  Every call has
    scratch of its own: torch's allocator keeps it from other streams and from other graphs."""
    n = cache._sizes.get(key)
    if n is None:
        with torch.cuda.device(cache._index):
            n = entry(cache._ref, ref)
        if n == 0:
            L.check(1, name)
        cache._sizes[key] = n
    return n


class PagedCache:
    """A batch of sequences over a pool of pages.

    k, v (n_pages, Hkv, page_size, D): the pool, float32 or bfloat16, D 64 or 128, any strides
    that are multiples of 16 bytes (last dimension contiguous; no strides of zero where rows are
    written).  table (batch, width) int32: slot j of sequence b lies in page
    ``table[b, j // page_size]`` at row ``j % page_size``; entries past a sequence's last page are
    not read.  lens (batch,) int32: tokens each sequence holds.
    weights (n_pages, Hkv, page_size) float32, optional: the attention weight that each key has
    received so far (``decode(weights_out=...)``), which ``evict`` ranks by.

    Keys, values and queries are finite numbers where a sequence has tokens; what a head gives that
    reads an infinity or NaN there is not defined (NaN, as a rule).  What lies in slots without a
    token is never read.

    The tensors are used in place and may be written by the program between calls (new table
    entries, new lengths); the object itself only keeps them and their addresses, so they are
    read-only attributes (another table or other lengths: ``with_pages``) and their storage must
    not be exchanged (``resize_``, ``set_``).  A page number outside the pool never faults: its
    sequence's result is NaN, its rows are dropped, and ``core.device_error()`` (of the cache's
    device) is 201 (append), 202 (decode) or 203 (evict).  Make the table no wider than the longest
    sequence needs (``with_pages`` on a slice): the scratch of ``decode`` with weights and the time
    of ``evict`` follow its width."""

    __slots__ = ("_tensors", "_index", "_args", "_ref", "_sizes", "_scale")

    k = property(lambda self: self._tensors[0])
    v = property(lambda self: self._tensors[1])
    table = property(lambda self: self._tensors[2])
    lens = property(lambda self: self._tensors[3])
    weights = property(lambda self: self._tensors[4])
    device = property(lambda self: self._tensors[5])

    def __init__(self, k, v, table, lens, weights=None):
        if not (torch.is_tensor(k) and k.is_cuda):
            raise ValueError("the cache must hold CUDA tensors (there is no CPU path)")
        if k.dim() != 4:
            raise ValueError("k, v must be (n_pages, Hkv, page_size, D)")
        dev = k.device
        code = dtype_code(k.dtype)
        _on(k, dev, k.dtype, k.shape, "k")
        _on(v, dev, k.dtype, k.shape, "v")
        _on(table, dev, torch.int32, (None, None), "table")
        _on(lens, dev, torch.int32, (table.shape[0],), "lens")
        n_pages, hk, page, d = k.shape
        if weights is not None:
            _on(weights, dev, torch.float32, (n_pages, hk, page), "weights")
        self._tensors = (k, v, table, lens, weights, dev)
        a = L.PagedCacheArgs()
        a.k, a.k_stride_p, a.k_stride_h, a.k_stride_n = k.data_ptr(), k.stride(0), k.stride(1), k.stride(2)
        a.v, a.v_stride_p, a.v_stride_h, a.v_stride_n = v.data_ptr(), v.stride(0), v.stride(1), v.stride(2)
        if weights is not None:
            a.weights, a.weights_stride_p, a.weights_stride_h = weights.data_ptr(), weights.stride(0), weights.stride(1)
        a.table, a.table_stride, a.lens = table.data_ptr(), table.stride(0), lens.data_ptr()
        a.dtype, a.d = code, d
        a.n_pages, a.n_kv_heads, a.page_size = n_pages, hk, page
        a.batch, a.table_width = table.shape
        self._args, self._ref, self._sizes = a, ctypes.byref(a), {}
        self._index, self._scale = dev.index, 1.0 / math.sqrt(d)

    @property
    def batch(self):
        return self.table.shape[0]

    def with_pages(self, table, lens):
        """The same pool under other page tables / lengths."""
        return PagedCache(self.k, self.v, table, lens, weights=self.weights)

    def _moved(self, table, lens):
        """with_pages for a table (of the same batch) and lengths that have been checked."""
        c = PagedCache.__new__(PagedCache)
        k, v, _, _, weights, dev = self._tensors
        c._tensors = (k, v, table, lens, weights, dev)
        a = L.PagedCacheArgs.from_buffer_copy(self._args)
        a.table, a.lens = table.data_ptr(), lens.data_ptr()
        a.table_stride, a.table_width = table.stride(0), table.shape[1]
        c._args, c._ref, c._sizes = a, ctypes.byref(a), {}
        c._index, c._scale = self._index, self._scale
        return c


def append(cache: PagedCache, k, v, *, counts=None, lens_out=None):
    """Write the first ``counts[b]`` of the rows k, v (batch, Hkv, n, D) to slots ``lens[b]`` on of
    sequence b (counts None: all n; a decode step has n = 1), set their weights to zero, and
    return the new lengths in ``lens_out`` (batch,) int32 (default: the cache's own ``lens``; it may
    be ``counts``).
    The caller has put pages for the new slots into the table; rows past its last slot are
    dropped and reported by ``core.device_error()``.  A page that is written must belong to one
    sequence alone (a shared page that is partly filled is copied first), and k, v must not lie
    where the call writes.  The weights stay zero until ``decode`` adds to them: evicted before
    that, a prompt is ranked by slot alone."""
    a = cache._args
    pool, _, _, lens, _, dev = cache._tensors
    if not (isinstance(k, torch.Tensor) and isinstance(v, torch.Tensor)):
        raise ValueError("k and v must be tensors")
    shape = (a.batch, a.n_kv_heads, k.shape[2] if k.dim() == 4 else None, a.d)
    if k.dim() == 4 and k.stride(3) != 1:
        k = k.contiguous()
    if v.dim() == 4 and v.stride(3) != 1:
        v = v.contiguous()
    dt = pool.dtype
    if not (k.shape == shape and v.shape == shape and k.dtype is dt and v.dtype is dt
            and k.device == dev and v.device == dev):
        _on(k, dev, dt, shape, "k")
        _on(v, dev, dt, shape, "v")
    if counts is not None:
        _on(counts, dev, torch.int32, (a.batch,), "counts")
    if lens_out is None:
        lens_out = lens
    else:
        _on(lens_out, dev, torch.int32, (a.batch,), "lens_out")
    kb, kh, kn, _ = k.stride()
    vb, vh, vn, _ = v.stride()
    b = L.PagedAppendArgs(k.data_ptr(), kb, kh, kn, v.data_ptr(), vb, vh, vn, shape[2],
                          None if counts is None else counts.data_ptr(), lens_out.data_ptr())
    _run(cache, L.lib().sta_paged_append, "sta_paged_append", ctypes.byref(b))
    return lens_out


def decode(q, cache: PagedCache, geometry: Geometry, *, sm_scale=None, weights_out=None):
    """Attention of one new token per sequence, q (batch, H, D) at position ``lens[b] - 1`` (its
    own key and value appended before), over all slots of its sequence.  ``geometry`` gives the
    positions: ``pos_scale`` and ``rope_scale``, or ``dca`` = (chunk_size, local_window) with a
    chunk length that is a multiple of 64.  Returns out (batch, H, D); a sequence of length 0
    gives zeros.  The same call gives the same bits; a sequence's last bits may depend on the lengths
    of the others in the batch.

    With ``weights_out`` (a tensor with the shape and strides of the cache's ``weights`` that does
    not overlap them, or the weights themselves) every slot receives its weight plus the attention weight that this token
    gave it, summed over the q heads of its kv head.  No page may stand in the table twice then
    (among the entries in use): one of its places adds its weights, the others' are dropped, and
    ``core.device_error()`` is 204.  In a bfloat16 cache an added weight is off by up to
    6 * 2^-16 |q| |k| sm_scale rope_scale^2 relative to itself (scores over a range of 8: 4e-6 in norm);
    a float32 cache gives fp32."""
    a = cache._args
    pool, _, _, _, weights, dev = cache._tensors
    _on(q, dev, pool.dtype, (a.batch, None, a.d), "q")
    inv = geometry.inv_freq
    if inv.dtype is not torch.float32 or inv.device != dev or not inv.is_contiguous():
        if inv.device != dev and torch.cuda.is_current_stream_capturing():
            raise ValueError(f"inv_freq must lie on {dev} where decode is captured into a graph")
        inv = inv.to(device=dev, dtype=torch.float32).contiguous()
    if inv.numel() != a.d // 2:
        raise ValueError("inv_freq must have head_dim/2 entries")
    H = q.shape[1]
    out = torch.empty_like(q, memory_format=torch.contiguous_format)
    qb, qh, _ = q.stride()
    b = L.PagedDecodeArgs(q.data_ptr(), qb, qh, out.data_ptr(), H, inv.data_ptr(),
                          float(geometry.pos_scale), float(geometry.rope_scale),
                          cache._scale if sm_scale is None else float(sm_scale))
    if geometry.dca is not None:
        size, window = int(geometry.dca[0]), int(geometry.dca[1])
        if window <= 0 or size <= window or (size - window) % 64 or size >= 1 << 31:
            raise ValueError(f"dca {size, window}: chunk_size - local_window must be a positive multiple of 64"
                             " (and chunk_size below 2^31)")
        b.chunk_size, b.local_window = size, window
    if weights_out is not None:
        if weights is None:
            raise ValueError("weights_out needs a cache with weights")
        _on(weights_out, dev, torch.float32, weights.shape, "weights_out")
        if weights_out.stride() != weights.stride():
            raise ValueError("weights_out must have the strides of the cache's weights")
        b.weights_out = weights_out.data_ptr()
    ref = ctypes.byref(b)
    lib = L.lib()
    n = _size(cache, (H, weights_out is None), lib.sta_paged_decode_workspace_bytes, "sta_paged_decode", ref)
    ws = torch.empty(n, dtype=torch.uint8, device=dev)
    _run(cache, lib.sta_paged_decode, "sta_paged_decode", ref, ws.data_ptr(), n)
    return out


def evict(cache: PagedCache, budget: int, table_out, *, n_global=32, n_local=32):
    """Cut every sequence to at most ``budget`` keys per kv head: the first ``n_global``, the last
    ``n_local``, and of the others those with the largest ``weights`` (ties: lowest slot).  The
    kept rows of k, v and weights are copied, in order, into the pages of ``table_out`` (batch,
    >= ceil(min(budget, slots) / page_size)) int32; the old pages stay as they are (they may be
    shared) until the caller frees them.  The new pages that are filled must all be different and
    must not be in use by the cache: of a page that two entries name one entry's rows are written,
    of a page in use none, the other rows are dropped, and ``core.device_error()`` is 204.

    Returns (the cache over the new pages, kept (batch, Hkv, budget) int32: the original slots in
    order, -1 beyond a sequence's new length)."""
    a = cache._args
    dev = cache._tensors[5]
    budget = int(budget)
    _on(table_out, dev, torch.int32, (a.batch, None), "table_out")
    if budget <= 0:
        raise ValueError("budget must be positive")
    kept = table_out.new_empty((a.batch, a.n_kv_heads, budget))
    lens = table_out.new_empty((a.batch,))
    b = L.PagedEvictArgs(budget, int(n_global), int(n_local), table_out.data_ptr(),
                         table_out.stride(0), table_out.shape[1], kept.data_ptr(), lens.data_ptr())
    ref = ctypes.byref(b)
    lib = L.lib()
    n = _size(cache, (budget, n_global, n_local, b.table_out_width), lib.sta_paged_evict_workspace_bytes,
              "sta_paged_evict", ref)
    ws = torch.empty(n, dtype=torch.uint8, device=dev)
    _run(cache, lib.sta_paged_evict, "sta_paged_evict", ref, ws.data_ptr(), n)
    return cache._moved(table_out, lens), kept
