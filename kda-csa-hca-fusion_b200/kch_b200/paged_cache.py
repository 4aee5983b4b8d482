"""A paged key / value cache for softmax attention beside the stack's own layers.

Not in the reference, whose decode caches hold one batch that advances in lock step (ops_decoding_cache.py:407-1395).
Here sequences of any lengths share a pool of pages and a call: some bring a chunk of a prompt, some one token.  The
caller assigns pages (a block table per batch); everything the kernels need of the lengths stays on the device, so a
captured CUDA graph replays with other lengths and tables.  ``kv_quant='fp8'|'int8'`` stores rows in 8 bits with one fp32
scale a row and key head, quantised as they are written.  Forward only.
"""
from __future__ import annotations

import torch

from . import _lib
from .decoding_cache import _QUANT, _validate_cache_dtype

_PAYLOAD = {"fp8": torch.float8_e4m3fn, "int8": torch.int8}


def _int_at_least(name, v, least):
    if not isinstance(v, int) or isinstance(v, bool) or v < least:
        raise ValueError(f"PagedKVCache: {name}={v!r} must be an int >= {least}")


def _packed(x):
    """``(tensor, its address, elements between tokens)`` of ``x [N, heads, c]`` whose heads are dense within a token (a column
    slice of a fused projection, say), copied where they are not, or not on 16 bytes."""
    N, heads, c = x.shape
    width, at = heads * c, x.data_ptr()
    if at % 16 == 0:
        if x.is_contiguous():
            return x, at, width
        token, head, inner = x.stride()
        if (c == 1 or inner == 1) and (heads == 1 or head == c) and (N <= 1 or (token >= width and token * x.element_size() % 16 == 0)):
            return x, at, token if N > 1 else width
    x = x.contiguous()
    if x.data_ptr() % 16:
        x = x.clone()
    return x, x.data_ptr(), width


class PagedKVCache:
    """``num_pages`` pages of ``page_size`` tokens for ``n_kv`` key heads of width ``c``.

    ``k_pages``, ``v_pages`` ``[num_pages, n_kv, page_size, c]`` in ``dtype`` (fp32 or bf16), or with ``kv_quant`` in e4m3 /
    int8 beside ``k_scales``, ``v_scales`` fp32 ``[num_pages, n_kv, page_size]``.  ``storage``: those four tensors of a pool
    that exists already (the scales None without ``kv_quant``).

    Every method takes a ragged batch of B sequences (at most 4096): ``table`` int32 ``[B, max_pages]``, ``t0`` int32 ``[B]``
    (tokens of a sequence before this call's) and ``cu_seqlens`` int32 ``[B + 1]``: rows ``cu_seqlens[b] .. cu_seqlens[b+1]`` of
    the packed tensors are the positions ``t0[b], t0[b] + 1, ..`` of sequence b, and position p lies in row ``p % page_size``
    of page ``table[b, p // page_size]``.  A table that names no page of the pool where one is needed, or ends before its
    sequence does, and a negative ``t0`` raise the device status ``KCH_STATUS_PAGED_TABLE``.
    """

    def __init__(self, num_pages, page_size, n_kv, c, device, dtype, *, kv_quant=None, storage=None):
        _int_at_least("num_pages", num_pages, 1)
        _int_at_least("page_size", page_size, 8)
        _int_at_least("n_kv", n_kv, 1)
        _int_at_least("c", c, 8)
        if num_pages > 0x7FFFFFFF:
            raise ValueError(f"PagedKVCache: num_pages={num_pages} does not fit a table of 32-bit page numbers")
        if page_size > 256 or page_size & (page_size - 1):
            raise ValueError(f"PagedKVCache: page_size={page_size} must be a power of two from 8 to 256")
        if c > 256 or c % 8:
            raise ValueError(f"PagedKVCache: c={c} must be a multiple of 8 from 8 to 256")
        _validate_cache_dtype(dtype)
        if kv_quant not in _QUANT:
            raise ValueError(f"kv_quant={kv_quant!r} must be one of {list(_QUANT)}")
        device = torch.device(device)
        if device.type != "cuda":
            raise RuntimeError(f"PagedKVCache: backend 'b200' requires a CUDA device, got {device}")
        self.num_pages, self.page_size, self.n_kv, self.c = num_pages, page_size, n_kv, c
        self.dtype, self.kv_quant = dtype, kv_quant
        shape = (num_pages, n_kv, page_size, c)
        payload = dtype if kv_quant is None else _PAYLOAD[kv_quant]
        if storage is None:
            k, v = (torch.zeros(shape, dtype=torch.uint8 if kv_quant else dtype, device=device) for _ in range(2))
            ks, vs = (torch.ones(shape[:3], dtype=torch.float32, device=device) if kv_quant else None for _ in range(2))
            storage = (k.view(payload), v.view(payload), ks, vs)
        if not isinstance(storage, (tuple, list)) or len(storage) != 4:
            raise ValueError("PagedKVCache: storage must be (k_pages, v_pages, k_scales, v_scales)")
        scale = None if kv_quant is None else torch.float32
        for name, t, want, dt in zip(("k_pages", "v_pages", "k_scales", "v_scales"), storage, (shape, shape, shape[:3], shape[:3]),
                                     (payload, payload, scale, scale)):
            if dt is None and t is not None:
                raise ValueError(f"PagedKVCache: {name} goes with kv_quant")
            if dt is not None and (not isinstance(t, torch.Tensor) or tuple(t.shape) != want or t.dtype != dt or not t.is_contiguous()):
                raise ValueError(f"PagedKVCache: {name} must be a contiguous {dt} tensor of shape {want}, got "
                                 f"{(tuple(t.shape), t.dtype) if isinstance(t, torch.Tensor) else t!r}")
        where = storage[0].device if device.index is None else device
        for name, t in zip(("k_pages", "v_pages", "k_scales", "v_scales"), storage):
            if t is not None and (t.device != where or not t.is_cuda):
                raise ValueError(f"PagedKVCache: {name} is on {t.device}, {where if where.type == 'cuda' else 'a CUDA device'} is expected")
            if t is not None and t.data_ptr() % 16:
                raise ValueError(f"PagedKVCache: {name} must start on 16 bytes")
        self.device = where
        self._storage = tuple(storage)
        self._ws_bytes = {}             # of attention calls, by their sizes
        self._row = torch.empty(0, dtype=dtype, device=self.device)        # (what new tensors are made from)
        self._byte = torch.empty(0, dtype=torch.uint8, device=self.device)
        self._tag, self._index, self._lib = _lib.dtype_tag(dtype), self.k_pages.get_device(), _lib.load()
        self._c = _lib.PagedCache(self.k_pages.data_ptr(), self.v_pages.data_ptr(), _lib.ptr(self.k_scales), _lib.ptr(self.v_scales),
                                  self._tag if kv_quant is None else _QUANT[kv_quant], num_pages, page_size, n_kv, c)

    # (not to be set: the kernels have their addresses)
    k_pages = property(lambda self: self._storage[0])
    v_pages = property(lambda self: self._storage[1])
    k_scales = property(lambda self: self._storage[2])
    v_scales = property(lambda self: self._storage[3])

    # A call of a decode step takes the host longer than the GPU: the checks compare what they can in one expression, and name
    # the argument at fault only where it fails.
    def _batch(self, fn, table, t0, cu_seqlens, N):
        shape, i32, index = table.shape, torch.int32, self._index
        if not (len(shape) == 2 and table.dtype is t0.dtype is cu_seqlens.dtype is i32 and table.get_device() == index == t0.get_device()
                and cu_seqlens.get_device() == index and t0.shape == shape[:1] and cu_seqlens.shape == (shape[0] + 1,)
                and 1 <= shape[0] <= 4096 and shape[1] >= 1):
            self._batch_error(fn, table, t0, cu_seqlens)
        B, P = shape
        ld, inner = table.stride()
        if (inner != 1 and P > 1) or (ld < P and B > 1):
            table = table.contiguous()
            ld = P
        if not t0.is_contiguous():
            t0 = t0.contiguous()
        if not cu_seqlens.is_contiguous():
            cu_seqlens = cu_seqlens.contiguous()
        return (_lib.PagedBatch(table.data_ptr(), ld if B > 1 else P, P, t0.data_ptr(), cu_seqlens.data_ptr(), B, N),
                (table, t0, cu_seqlens))

    def _batch_error(self, fn, table, t0, cu_seqlens):
        for name, t, rank in (("table", table, 2), ("t0", t0, 1), ("cu_seqlens", cu_seqlens, 1)):
            if t.dim() != rank:
                raise ValueError(f"{fn}: {name} must have rank {rank}, got shape {tuple(t.shape)}")
            if t.dtype != torch.int32:
                raise TypeError(f"{fn}: {name} must be int32, got {t.dtype}")
            if t.device != self.device:
                raise ValueError(f"{fn}: {name} is on {t.device}, the cache on {self.device}")
        B = table.shape[0]
        if not 1 <= B <= 4096:
            raise ValueError(f"{fn}: {B} sequences; a call takes 1 to 4096")
        if table.shape[1] < 1:
            raise ValueError(f"{fn}: table has no columns")
        raise ValueError(f"{fn}: t0 {tuple(t0.shape)} and cu_seqlens {tuple(cu_seqlens.shape)} must have {B} and {B + 1} entries")

    def _rows(self, fn, name, x, heads=None):
        shape = x.shape
        if len(shape) == 3 and shape[2] == self.c and (heads is None or shape[1] == heads) and x.dtype is self.dtype \
                and x.get_device() == self._index:
            return shape
        if x.dim() != 3 or shape[2] != self.c or (heads is not None and shape[1] != heads):
            raise ValueError(f"{fn}: {name} must be [N, {'nh' if heads is None else heads}, {self.c}], got {tuple(shape)}")
        if x.dtype != self.dtype:
            raise ValueError(f"{fn}: {name}.dtype={x.dtype} does not match the cache's {self.dtype}")
        raise (ValueError if x.is_cuda else RuntimeError)(f"{fn}: {name} is on {x.device}, the CUDA cache on {self.device}")

    def _own_out(self, fn, name, x, shape):
        self._rows(fn, name, x, shape[1])
        if x.shape[0] != shape[0] or not x.is_contiguous() or x.data_ptr() % 16:
            raise ValueError(f"{fn}: {name} must be a contiguous {tuple(shape)} tensor on 16 bytes, got {tuple(x.shape)}")

    def append_step(self, k_new, v_new, table, t0, cu_seqlens):
        """Writes the new rows ``k_new``, ``v_new`` ``[N, n_kv, c]`` into their pages.  Rows outside of
        ``[cu_seqlens[0], cu_seqlens[B])`` are not read.  No two rows of a call go to one place of the pool (pages that sequences
        share hold tokens before the call's)."""
        fn = "append_step"
        N = self._rows(fn, "k_new", k_new, self.n_kv)[0]
        if self._rows(fn, "v_new", v_new, self.n_kv)[0] != N:
            raise ValueError(f"{fn}: v_new has {v_new.shape[0]} rows, k_new {N}")
        batch, keep = self._batch(fn, table, t0, cu_seqlens, N)
        with _lib.device(self.device):
            k, at_k, ld_k = _packed(k_new)
            v, at_v, ld_v = _packed(v_new)
            _lib.check(self._lib.kch_paged_append(self._c, batch, at_k, ld_k, at_v, ld_v, self._tag, _lib.stream()))

    def read_step(self, table, t0, cu_seqlens, *, n_rows, out=None):
        """The rows of those positions as ``(k, v)`` ``[n_rows, n_kv, c]`` in the cache's ``dtype`` (stored value times scale).
        ``n_rows`` is ``cu_seqlens[B]``, which only the device knows, or more: rows of no sequence are zeros, and stay as they
        are in tensors given as ``out``."""
        fn = "read_step"
        _int_at_least("n_rows", n_rows, 0)
        shape = (n_rows, self.n_kv, self.c)
        batch, keep = self._batch(fn, table, t0, cu_seqlens, n_rows)
        with _lib.device(self.device):
            if out is None:
                k, v = self._row.new_empty(shape), self._row.new_empty(shape)
            else:
                k, v = out
                self._own_out(fn, "out[0]", k, shape)
                self._own_out(fn, "out[1]", v, shape)
            width = self.n_kv * self.c
            _lib.check(self._lib.kch_paged_read(self._c, batch, k.data_ptr(), width, v.data_ptr(), width, self._tag, int(out is None),
                                                  _lib.stream()))
        return k, v

    def forward_step(self, q, table, t0, cu_seqlens, *, scale=None, sink_logits=None, sliding_window=0, out=None):
        """Attention of the batch's new tokens, whose own rows :meth:`append_step` has written: ``q [N, nh, c]`` (``nh`` a
        multiple of ``n_kv``; query head h reads key head ``h // (nh // n_kv)``) -> ``[N, nh, c]`` in ``q.dtype``.  The query at
        position p sees the keys ``0 .. p``, or the last ``sliding_window`` of them (entries of pages that no query of a sequence
        reaches any more are not used).  ``scale``: ``c ** -0.5`` unless given;
        ``sink_logits [nh]`` adds ``exp(sink)`` to the denominator.  Rows of no sequence are zeros, and stay as they are in a
        tensor given as ``out``, which does not overlap ``q``."""
        fn = "forward_step"
        N, nh, c = self._rows(fn, "q", q)
        if nh < 1 or nh % self.n_kv:
            raise ValueError(f"{fn}: nh={nh} must be a multiple of n_kv={self.n_kv}")
        if not isinstance(sliding_window, int) or isinstance(sliding_window, bool) or sliding_window < 0:
            raise ValueError(f"{fn}: sliding_window={sliding_window!r} must be an int >= 0 (0: every key)")
        batch, keep = self._batch(fn, table, t0, cu_seqlens, N)
        with _lib.device(self.device):
            sink, sink_tag = None, 0
            if sink_logits is not None:
                if tuple(sink_logits.shape) != (nh,) or sink_logits.get_device() != self._index:
                    raise ValueError(f"{fn}: sink_logits must be [{nh}] on {self.device}, got {tuple(sink_logits.shape)} on {sink_logits.device}")
                sink_logits = sink_logits.contiguous()
                sink, sink_tag = sink_logits.data_ptr(), _lib.dtype_tag(sink_logits.dtype)
            q, at_q, ld_q = _packed(q)
            if out is None:
                o = self._row.new_empty((N, nh, c))
            else:
                o = out
                self._own_out(fn, "out", o, (N, nh, c))
            a = _lib.PagedAttendArgs(self._c, batch, at_q, ld_q, self._tag, nh, c ** -0.5 if scale is None else float(scale),
                                     min(sliding_window, 0x7FFFFFFF), sink, sink_tag, o.data_ptr(), int(out is None))
            sizes = (N, nh, batch.B)
            nbytes = self._ws_bytes.get(sizes)
            if nbytes is None:
                if len(self._ws_bytes) > 4096:
                    self._ws_bytes.clear()
                nbytes = self._ws_bytes[sizes] = int(self._lib.kch_paged_attend_workspace_bytes(a))
            ws = self._byte.new_empty(nbytes)
            a.workspace, a.workspace_bytes = ws.data_ptr(), nbytes
            _lib.check(self._lib.kch_paged_attend(a, _lib.stream()))
        return o
