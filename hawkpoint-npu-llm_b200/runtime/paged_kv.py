"""A paged K/V cache on the device, and the operators on it.

``PagedKVCache`` holds a pool of 64-position pages with its books (page table,
reference counts, lengths) in device memory and calls the paged operators of
libhawkb200.so (include/hawkb200.h) on torch tensors, on torch's current
stream: nothing here waits for the GPU or copies to the host, except
``status``.  The reference keeps one contiguous 64-position cache per process
(npu_llm/runtime/qwen_engine.py:65-94); the engine's own paged cache
(``B200DecoderEngine(context=...)``) keeps its books on the host.

A step of a serving loop, per layer the two calls in the middle::

    cache.reserve(slots, counts)                  # room for the new rows
    q = cache.append(layer, qkv, slots, row_start, max_rows, cos, sin)
    o = cache.attend(layer, q, slots, row_start, max_rows)
    cache.fork(src, dst, counts); cache.free(done); cache.compact()

Entry b of a call is slot ``slots[b]`` with rows ``row_start[b] ..
row_start[b + 1]``; its row i of n stands at position ``lengths[slot] - n + i``.
Rows before the first and after the last start give 0 (and -inf).
All index lists are int32 device tensors.  Pages are laid out
``[layer][kv head][K | V][head_dim / 64][64 positions][64 dims]`` with the
16-byte blocks of a position's 64 dims stored at block ^ (position & 7);
``rows`` gives a slot's K and V in plain order.

Calls on one cache share its workspace: run them on one stream, or order the
streams with events, and make them from one thread at a time.
"""

import ctypes
import struct

from runtime import hb_lib

PAGE = 64
_WIDEST = 2 ** 31 - 1   # a window's most; no context is longer

# The structs of a call, filled in place: a decode step makes tens of calls, and
# building ctypes objects for each would cost more than the launches.
_ROWS = struct.Struct("=QQiiii")            # hb_paged_rows
_QUERY = struct.Struct("=QqqQqqQiifi")      # hb_paged_query
_NEW = struct.Struct("=QqQqqQQii")          # hb_paged_new
assert (_ROWS.size, _QUERY.size, _NEW.size) == tuple(
    ctypes.sizeof(c) for c in (hb_lib.HbPagedRows, hb_lib.HbPagedQuery, hb_lib.HbPagedNew))


def _torch():
    import torch

    return torch


class PagedKVCache:
    """A pool of ``n_pages`` pages and its books for ``n_slots`` sequences of
    up to ``max_context`` positions (rounded up to whole pages)."""

    def __init__(self, layers, kv_heads, head_dim, n_pages, n_slots, max_context, dtype=None, device=None):
        torch = _torch()
        dtype = torch.bfloat16 if dtype is None else dtype
        device = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
        if min(layers, kv_heads, n_pages, n_slots, max_context) < 1:
            raise ValueError("layers, kv_heads, n_pages, n_slots and max_context must be positive")
        if head_dim not in (64, 128):
            raise ValueError(f"head_dim {head_dim}: must be 64 or 128")
        ints = dict(dtype=torch.int32, device=device)
        self._bind(torch.zeros((n_pages, layers, kv_heads, 2, head_dim // 64, PAGE, 64), dtype=dtype, device=device),
                   torch.full((n_slots, -(-max_context // PAGE)), -1, **ints), torch.zeros(n_pages, **ints),
                   torch.zeros(n_slots, **ints))

    @classmethod
    def wrap(cls, pool, table, refs, lengths):
        """A cache over the caller's tensors: ``pool`` [pages, layers, kv
        heads, 2, head_dim / 64, 64, 64] (pages may lie apart, a page's
        elements together), ``table`` int32 [slots, pages a slot], ``refs`` int32
        [pages], ``lengths`` int32 [slots]."""
        cache = cls.__new__(cls)
        cache._bind(pool, table, refs, lengths)
        return cache

    def _bind(self, pool, table, refs, lengths):
        torch = _torch()
        if pool.device.type != "cuda":   # the kernels would read host addresses
            raise ValueError(f"pool on {pool.device}: must be on a CUDA device")
        elements = {torch.bfloat16: hb_lib.HB_ELEM_BF16, torch.float16: hb_lib.HB_ELEM_FP16}
        if pool.dtype not in elements:
            raise ValueError(f"pool of {pool.dtype}: must be bfloat16 or float16")
        if pool.dim() != 7 or pool.shape[3] != 2 or tuple(pool.shape[5:]) != (PAGE, 64) or pool.shape[4] not in (1, 2):
            raise ValueError(f"pool of shape {tuple(pool.shape)}: must be [pages, layers, kv heads, 2, head_dim / 64, 64, 64]")
        if pool.shape[0] < 1 or not pool[0].is_contiguous():
            raise ValueError("a page's elements must be contiguous")
        n_pages, layers, kv_heads = (int(x) for x in pool.shape[:3])
        for name, t, shape in (("table", table, None), ("refs", refs, (n_pages,)), ("lengths", lengths, (table.shape[0],))):
            if t.dtype != torch.int32 or not t.is_contiguous() or t.device != pool.device:
                raise ValueError(f"{name} must be a contiguous int32 tensor on the pool's device")
            if shape is not None and tuple(t.shape) != shape:
                raise ValueError(f"{name} of shape {tuple(t.shape)}: must be {shape}")
        if table.dim() != 2:
            raise ValueError("table must have a row a slot")
        self._lib = hb_lib.load()
        self.pool, self.table, self.refs, self.lengths = pool, table, refs, lengths
        self.device, self.dtype = pool.device, pool.dtype
        self.layers, self.kv_heads, self.head_dim = layers, kv_heads, 64 * int(pool.shape[4])
        p = self._desc = hb_lib.HbPagePool(
            pages_dev=pool.data_ptr(), page_stride=pool.stride(0) * 2, n_pages=n_pages, layers=layers,
            kv_heads=kv_heads, head_dim=self.head_dim, element=elements[pool.dtype], n_slots=int(table.shape[0]),
            table_width=int(table.shape[1]), table_dev=table.data_ptr(), refs_dev=refs.data_ptr(),
            lengths_dev=lengths.data_ptr())
        if n_pages == 1:
            p.page_stride = pool[0].numel() * 2
        self._pool = ctypes.addressof(p)
        need = self._lib.hb_paged_workspace_bytes(self._pool)
        if need == 0:
            hb_lib.check(hb_lib.HB_ERR_INVALID_ARG)
        self._workspace = torch.zeros(need, dtype=torch.uint8, device=pool.device)
        p.workspace_dev, p.workspace_bytes = self._workspace.data_ptr(), need
        self._index = pool.device.index if pool.device.index is not None else torch.cuda.current_device()
        self._int32, self._float32 = torch.int32, torch.float32
        self._scale = self.head_dim ** -0.5
        self._empty = torch.empty_strided
        # the current device and the current stream's handle, by torch's own accessors where it has them
        self._current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)
        self._current_stream = getattr(torch._C, "_cuda_getCurrentRawStream",
                                       lambda index: torch.cuda.current_stream(index).cuda_stream)
        self._attend, self._append = self._lib.hb_paged_attend, self._lib.hb_paged_append
        # what a call fills, and its addresses
        self._rows_buf, self._args_buf = bytearray(_ROWS.size), bytearray(max(_QUERY.size, _NEW.size))
        self._rows_at, self._args_at = (ctypes.addressof(ctypes.c_char.from_buffer(b)) for b in (self._rows_buf, self._args_buf))

    # -- helpers -----------------------------------------------------------------
    def _call(self, fn, *args):
        if self._current_device() == self._index:
            rc = fn(self._pool, *args, self._current_stream(self._index))
        else:
            with _torch().cuda.device(self._index):
                rc = fn(self._pool, *args, self._current_stream(self._index))
        if rc:
            hb_lib.check(rc)

    def _list(self, name, t, n=None):
        if t.dtype is not self._int32 or t.dim() != 1 or not t.is_contiguous() or t.get_device() != self._index:
            raise ValueError(f"{name} must be a contiguous one-dimensional int32 tensor on the cache's device")
        if n is not None and t.numel() != n:
            raise ValueError(f"{name} has {t.numel()} entries, not {n}")
        return t.data_ptr()

    def _run(self, fn, layer, slots, row_start, rows, max_rows):
        entries = slots.numel()
        if not 0 <= layer < self.layers:   # ctypes would cut it to 32 bits
            raise ValueError(f"layer {layer} outside [0, {self.layers})")
        if max_rows < 0 or (entries == 0 and rows > 0):
            raise ValueError("max_rows must not be negative, and rows need an entry")
        _ROWS.pack_into(self._rows_buf, 0, self._list("slots", slots), self._list("row_start", row_start, entries + 1),
                        entries, rows, max_rows if max_rows < rows else rows, 0)
        index = self._index
        if self._current_device() != index:
            return self._call(fn, layer, self._rows_at, self._args_at)
        rc = fn(self._pool, layer, self._rows_at, self._args_at, self._current_stream(index))
        if rc:
            hb_lib.check(rc)

    def _heads(self, name, t, rows=None):
        """(shape, strides) of rows of heads."""
        if t.dtype is not self.dtype or t.dim() != 3 or t.get_device() != self._index:
            raise ValueError(f"{name} must be [rows, heads, {self.head_dim}] of {self.dtype} on the cache's device")
        shape, stride = t.shape, t.stride()
        if shape[2] != self.head_dim or stride[2] != 1:
            raise ValueError(f"{name} of shape {tuple(shape)}: its last dimension must be {self.head_dim}, contiguous")
        if rows is not None and shape[:2] != rows:
            raise ValueError(f"{name} of shape {tuple(shape)}: must be {tuple(rows) + (self.head_dim,)}")
        return shape, stride

    def _new_heads(self, rows, heads):
        d = self.head_dim
        return self._empty((rows, heads, d), (heads * d, d, 1), dtype=self.dtype, device=self.device)

    # -- rows ----------------------------------------------------------------------
    def append(self, layer, qkv, slots, row_start, max_rows, cos, sin, out=None):
        """Rotates the rows' q and k at their positions and stores k and v in
        the slots' pages (``reserve`` has mapped them).  ``qkv`` [rows, (q
        heads + 2 kv heads) * head_dim]; ``cos`` / ``sin`` float32 [positions,
        head_dim / 2].  Returns the rotated q [rows, q heads, head_dim]."""
        d = self.head_dim
        if qkv.dtype is not self.dtype or qkv.dim() != 2 or qkv.get_device() != self._index:
            raise ValueError(f"qkv must be [rows, heads * {d}] of {self.dtype} on the cache's device")
        (rows, cols), (row_stride, col_stride) = qkv.shape, qkv.stride()
        if cols % d or col_stride != 1:
            raise ValueError(f"qkv of shape {tuple(qkv.shape)}: its rows must be whole heads of {d}, contiguous")
        q_heads = cols // d - 2 * self.kv_heads
        if q_heads < 0:
            raise ValueError(f"qkv has fewer heads than the {2 * self.kv_heads} of k and v")
        table = cos.shape
        if len(table) != 2 or table[1] * 2 != d or sin.shape != table or (
                cos.dtype is not self._float32 or sin.dtype is not self._float32 or cos.get_device() != self._index
                or sin.get_device() != self._index or not (cos.is_contiguous() and sin.is_contiguous())):
            raise ValueError(f"cos and sin must be contiguous float32 [positions, {d // 2}] on the cache's device, of one "
                             "shape")
        if out is None:
            out, q_row, q_head = self._new_heads(rows, q_heads), q_heads * d, d
        else:
            _, (q_row, q_head, _) = self._heads("out", out, (rows, q_heads))
        _NEW.pack_into(self._args_buf, 0, qkv.data_ptr(), row_stride, out.data_ptr(), q_row, q_head, cos.data_ptr(),
                       sin.data_ptr(), table[0], q_heads)
        self._run(self._append, layer, slots, row_start, rows, max_rows)
        return out

    def attend(self, layer, q, slots, row_start, max_rows, scale=None, window=0, out=None, lse=False):
        """Attention of the rows' ``q`` [rows, q heads, head_dim] over their
        slots' positions up to each row's own (with ``window``: the last
        ``window`` of them); ``scale`` defaults to 1 / sqrt(head_dim).  Returns
        the output in q's shape; with ``lse`` also float32 [rows, q heads], the
        log of the sum of exp(scores).  Rows that see nothing give 0 and -inf.
        ``out`` must not overlap ``q``.  No gradient is recorded, whatever q
        requires."""
        (rows, heads, d), (q_row, q_head, _) = self._heads("q", q)
        if out is None:
            out, o_row, o_head = self._new_heads(rows, heads), heads * d, d
        else:
            _, (o_row, o_head, _) = self._heads("out", out, (rows, heads))
        sums = self._empty((rows, heads), (heads, 1), dtype=self._float32, device=self.device) if lse else None
        _QUERY.pack_into(self._args_buf, 0, q.data_ptr(), q_row, q_head, out.data_ptr(), o_row, o_head,
                         sums.data_ptr() if lse else 0, heads, window if window < _WIDEST else _WIDEST, self._scale if scale is None else scale, 0)
        self._run(self._attend, layer, slots, row_start, rows, max_rows)
        return (out, sums) if lse else out

    # -- pages -----------------------------------------------------------------------
    def reserve(self, slots, counts):
        """Room for ``counts[b]`` more positions of ``slots[b]``: lengths grow,
        missing pages are mapped (the lowest free ones), shared pages that
        will be written become the slot's own.  All or nothing (``status``)."""
        n = slots.shape[0]
        self._call(self._lib.hb_pages_reserve, n, self._list("slots", slots), self._list("counts", counts, n))

    def fork(self, src, dst, counts):
        """Slot ``dst[b]`` becomes the first ``counts[b]`` positions of
        ``src[b]`` as it was before the call; whole pages are shared."""
        n = src.shape[0]
        self._call(self._lib.hb_pages_fork, n, self._list("src", src), self._list("dst", dst, n),
                   self._list("counts", counts, n))

    def free(self, slots):
        """The slots' pages go back to the pool; their lengths become 0."""
        self._call(self._lib.hb_pages_free, slots.shape[0], self._list("slots", slots))

    def compact(self):
        """Moves the pages in use to the pool's lowest indices; returns each
        page's new index, int32 [pages], -1 for a free one."""
        page_map = _torch().empty_like(self.refs)
        self._call(self._lib.hb_pages_compact, page_map.data_ptr())
        return page_map

    def copy_pages(self, src, dst, to=None):
        """Copies whole pages ``src[i]`` to ``dst[i]`` of this pool, or of the
        cache ``to`` of the same layout.  No books change."""
        n = src.shape[0]
        if to is not None and (to.pool.shape[1:] != self.pool.shape[1:] or to.dtype != self.dtype
                               or to.device != self.device or to._desc.page_stride != self._desc.page_stride):
            raise ValueError("the destination's pages must have this cache's layout")
        self._call(self._lib.hb_pages_copy, n, self._list("src", src), self._list("dst", dst, n),
                   to.pool.data_ptr() if to is not None else None, to._desc.n_pages if to is not None else 0)

    def status(self):
        """Waits for the stream and raises what the calls since the last
        status met on the device: ``HbTimeout``, or ``HbError`` for an
        exhausted pool, an index out of range or a row without a page."""
        self._call(lambda pool, stream: self._lib.hb_paged_status(pool, None, stream))

    def rows(self, layer, slot):
        """K and V of a slot's positions in plain order, [2, kv heads, length,
        head_dim] (diagnostics: reads the table on the host)."""
        torch = _torch()
        length = int(self.lengths[slot])
        pages = self.table[slot, : -(-length // PAGE)].long()
        if len(pages) * PAGE < length or bool(((pages < 0) | (pages >= self.pool.shape[0])).any()):
            raise ValueError(f"slot {slot} has no page for some of its {length} positions")
        x = self.pool[pages, layer].view(len(pages), self.kv_heads, 2, -1, PAGE, 8, 8)
        at = torch.arange(PAGE, device=self.device)[:, None]
        x = x[..., at, torch.arange(8, device=self.device)[None, :] ^ (at & 7), :]
        x = x.permute(2, 1, 0, 4, 3, 5, 6).reshape(2, self.kv_heads, -1, self.head_dim)
        return x[:, :, :length]
