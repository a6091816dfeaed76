"""A paged FP8 KV cache (include/ds4hip_pages.h).

`PagePool` holds pages of FP8 rows for all layers, the sequences' page tables
and the pages' reference counts, all on the device: sequences are extended,
forked (pages shared or copied), cut and freed, and the pool is compacted,
without a wait for the host. What a call finds wrong on the device (too few free
pages, a sequence that is not there) goes to `status`; `check()` reads it.
"""
from __future__ import annotations

import ctypes as C

import torch

from ._lib import Ds4HipError, call, lib
from .ops import (HEAD_DIM, N_NOPE, N_ROT, Fp8KVCache, WindowView, _addr, _check, _int32, _on_stream, _ptr, _ready, _same_gpu,
                  _stream)

MAX_JOBS = 1024    # sequences of one call


class KvPages(C.Structure):
    """ds4hip_kv_pages."""
    _fields_ = [("codes", C.c_void_p), ("sexp", C.c_void_p), ("tail", C.c_void_p), ("layer_rows", C.c_longlong),
                ("n_layers", C.c_int), ("n_pages", C.c_int), ("page_rows", C.c_int), ("table_stride", C.c_int),
                ("n_seqs", C.c_int), ("refs", C.c_void_p), ("table", C.c_void_p), ("rows", C.c_void_p),
                ("status", C.c_void_p)]


class PagePool:
    """Pages of `page_rows` rows (a power of two) for every layer.

    codes uint8 [layers, pages * page_rows, 448], sexp int8 [.., 8], tail f16 (or
    its bits) [.., 64]; refs int32 [pages], table int32 [sequences, entries], rows
    int32 [sequences]. The pool works on these tensors; entries of `table` past a
    sequence's rows have no meaning. Calls on one pool are ordered on one stream.
    """

    def __init__(self, codes, sexp, tail, refs, table, rows, page_rows, status=None):
        if codes.dim() != 3 or table.dim() != 2:
            raise Ds4HipError("codes must be [layers, rows, 448] and table [sequences, entries]", -22)
        if len({t.device for t in (codes, sexp, tail, refs, table, rows, codes if status is None else status)}) > 1:
            raise Ds4HipError("the pool's tensors must be on one device", -22)
        layers, n_rows = codes.shape[0], codes.shape[1]
        n_pages = refs.numel()
        _check(codes, torch.uint8, layers * n_rows * N_NOPE, "codes")
        _check(sexp, torch.int8, layers * n_rows * 8, "sexp")
        _check(tail, tail.dtype, layers * n_rows * N_ROT, "tail")
        _check(refs, torch.int32, None, "refs")
        _check(table, torch.int32, None, "table")
        _check(rows, torch.int32, table.shape[0], "rows")
        if codes.shape[2] != N_NOPE or tail.element_size() != 2 or n_rows != n_pages * int(page_rows):
            raise Ds4HipError("codes, tail or refs do not fit pages of that many rows", -22)
        with torch.cuda.device(codes.device):
            self.status = torch.zeros(1, dtype=torch.int32, device=codes.device) if status is None else status
        _check(self.status, torch.int32, 1, "status")
        self.codes, self.sexp, self.tail = codes, sexp, tail
        self.refs, self.table, self.rows = refs, table, rows
        self.page_rows, self.n_layers, self.n_pages, self.n_seqs = int(page_rows), layers, n_pages, table.shape[0]
        self.device, self.index = codes.device, codes.device.index
        for n, name in ((layers, "codes"), (n_pages, "refs"), (self.page_rows, "page_rows"), (table.shape[1], "table"),
                        (self.n_seqs, "table")):
            _int32(n, name)
        self.c = KvPages(_ptr(codes), _ptr(sexp), _ptr(tail), n_rows, layers, n_pages, self.page_rows, table.shape[1],
                         self.n_seqs, _ptr(refs), _ptr(table), _ptr(rows), _ptr(self.status))
        self._c = C.byref(self.c)
        self._workspace = None
        self._views = {}

    @classmethod
    def empty(cls, n_pages, page_rows, n_seqs, max_rows, n_layers=1, device="cuda"):
        """A pool with every page free, for sequences of up to max_rows rows."""
        n = n_pages * page_rows
        pool = cls(torch.zeros((n_layers, n, N_NOPE), dtype=torch.uint8, device=device),
                   torch.zeros((n_layers, n, 8), dtype=torch.int8, device=device),
                   torch.zeros((n_layers, n, N_ROT), dtype=torch.int16, device=device),
                   torch.empty(n_pages, dtype=torch.int32, device=device),
                   torch.empty((n_seqs, -(-max_rows // page_rows)), dtype=torch.int32, device=device),
                   torch.empty(n_seqs, dtype=torch.int32, device=device), page_rows)
        with torch.cuda.device(pool.device):
            call("ds4hip_kv_pages_init", pool._c, _stream(None))
        return pool

    def layer(self, layer) -> Fp8KVCache:
        """The rows of one layer, as the other FP8 launchers take them."""
        return Fp8KVCache(self.codes[layer], self.sexp[layer], self.tail[layer])

    def check(self):
        """Waits for the device; raises Ds4HipError where a call was refused there
        since the last check (-22 or -28), and resets the status."""
        torch.cuda.synchronize(self.device)   # (whatever stream the calls were made on)
        code = int(self.status.item())
        if code:
            self.status.zero_()
            torch.cuda.synchronize(self.device)
            raise Ds4HipError("PagePool", code)

    def _jobs(self, ids, name, n=None):
        if ids is None:
            return 0
        if not _ready(ids, torch.int32, self.index):
            _check(ids, torch.int32, None, name)
            _same_gpu(ids, self.index, name)
        k = ids.numel()
        if n is not None and k != n:
            raise Ds4HipError(f"{name}: {n} entries expected, got {k}", -22)
        if k > MAX_JOBS:
            raise Ds4HipError(f"{name}: a call takes {MAX_JOBS} sequences at most, got {k}", -22)
        return k

    def _call(self, name, stream, *args):
        with _on_stream(stream, self.device):
            call(name, self._c, *args, _stream(stream))

    def _empty(self, size, dtype, stream):
        with _on_stream(stream, self.device):
            return torch.empty(size, dtype=dtype, device=self.device)

    def _ws(self, stream):
        if self._workspace is None:
            need = lib().ds4hip_kv_pages_workspace_bytes(self._c)
            self._workspace = self._empty(need, torch.uint8, stream)
            self._ws_args = (self._workspace.data_ptr(), need)
        return self._ws_args

    def extend(self, seqs, n_new, n_dst, dst_rows=None, stream=None):
        """n_new[j] more rows for sequence seqs[j] (int32 device tensors): takes the
        lowest free pages and returns the rows' places, int64 [n_dst], job after job
        (-1 past the last job's rows, or everywhere where the call is refused)."""
        n = self._jobs(seqs, "seqs")
        self._jobs(n_new, "n_new", n)
        n_dst = _int32(n_dst, "n_dst")
        if dst_rows is None:
            dst_rows = self._empty(n_dst, torch.int64, stream)
        else:
            _check(dst_rows, torch.int64, n_dst, "dst_rows")
            _same_gpu(dst_rows, self.index, "dst_rows")
        self._call("ds4hip_kv_pages_extend", stream, _addr(seqs), _addr(n_new), n, dst_rows.data_ptr(), n_dst)
        return dst_rows

    def append(self, kv, dst_rows, layer=0, stream=None):
        """Quantizes fp32 rows kv [n, 512] into the layer at dst_rows (extend's); a row
        whose place is -1 is skipped."""
        n, layer = _int32(kv.shape[0], "kv"), _int32(layer, "layer")
        _check(kv, torch.float32, n * HEAD_DIM, "kv")
        _check(dst_rows, torch.int64, n, "dst_rows")
        _same_gpu(kv, self.index, "kv")
        _same_gpu(dst_rows, self.index, "dst_rows")
        self._call("ds4hip_kv_pages_append", stream, layer, kv.data_ptr(), n, dst_rows.data_ptr())

    def fork(self, parents, children, n_rows=None, deep=False, stream=None):
        """children[j] (empty sequences) become copies of the first n_rows[j] rows (None
        or negative: all) of parents[j]: full pages shared and a partly filled last page
        copied, or every page copied (deep)."""
        n = self._jobs(parents, "parents")
        self._jobs(children, "children", n)
        self._jobs(n_rows, "n_rows", n)
        self._call("ds4hip_kv_pages_fork", stream, _addr(parents), _addr(children), _addr(n_rows), n, int(bool(deep)),
                   *self._ws(stream))

    def free(self, seqs, keep=None, stream=None):
        """Cuts sequences seqs[j] down to keep[j] rows (None: to nothing) and releases
        their other pages."""
        n = self._jobs(seqs, "seqs")
        self._jobs(keep, "keep", n)
        self._call("ds4hip_kv_pages_free", stream, _addr(seqs), _addr(keep), n)

    def compact(self, n_live=None, stream=None):
        """Moves the held pages to the front of the pool; returns their number, an int32
        device scalar."""
        if n_live is None:
            n_live = self._empty((), torch.int32, stream)
        else:
            _check(n_live, torch.int32, 1, "n_live")
            _same_gpu(n_live, self.index, "n_live")
        self._call("ds4hip_kv_pages_compact", stream, n_live.data_ptr(), *self._ws(stream))
        return n_live

    def attend(self, q, *, seqs=None, q_start=None, window=0, n_first=0, sinks=None, layer=0, out=None, workspace=None,
               stream=None):
        """ops.flash_attn_window_fp8 over this pool's pages of one layer: the sequences
        seqs (None: slots 0, 1, ..). Queries that q_start names for none of them are left
        as they were in out, and undefined without out."""
        view = self._views.get(layer)
        if view is None:
            view = self._views[layer] = WindowView(self.layer(layer), self.table, self.rows, self.page_rows)
        return view.attend(q, window=window, n_first=n_first, sinks=sinks, q_start=q_start, seq_ids=seqs, out=out,
                           workspace=workspace, stream=stream)
