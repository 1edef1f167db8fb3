"""Pages of a KV cache that several sequences hold at once (``tq_pages_*`` in include/tangq.h): forked sequences share their
pages, and a shared page is copied when one of them is about to write it.  All bookkeeping happens on the device, so that the
calls can be recorded in a graph (with lists that are Buffers); ``state()`` is the only one that waits."""
from __future__ import annotations

import ctypes as C

import numpy as np

from . import _lib
from ._lib import TQ_EINVAL, TangqError
from .device import Buffer, QuantComputeDevice, _opt_ptr


class PagePool:
    """`n_pages` pages of `page_rows` positions (16, 32, .. 1024) for `n_seqs` sequences with at most `max_pages` each.

    `arrays`: the caches that the pages are cut from, one Buffer of [n_pages][page_rows][row] for the keys and one for the values
    of every layer.  `refs` / `tables` / `lens`: int32 Buffers [n_pages], [n_seqs][max_pages], [n_seqs] of the caller's with the
    pool's state; without them the pool has its own and starts empty."""

    def __init__(self, dev: QuantComputeDevice, n_pages: int, page_rows: int, n_seqs: int, max_pages: int, arrays=None, refs: Buffer | None = None,
                 tables: Buffer | None = None, lens: Buffer | None = None):
        self.dev, self.n_pages, self.page_rows, self.n_seqs, self.max_pages, self.handle = dev, n_pages, page_rows, n_seqs, max_pages, 0
        for b, n in ((refs, n_pages), (tables, n_seqs * max_pages), (lens, n_seqs)):
            if b is not None and (b.n != n or b.dtype != _lib.I32):
                raise TangqError(TQ_EINVAL, f"PagePool: {b.n} values of state where {n} of int32 are needed")
        self._keep = [refs, tables, lens]
        h = C.c_void_p()
        dev._check(dev._L.tq_pages_create(dev._ctx, n_pages, page_rows, n_seqs, max_pages, _opt_ptr(refs), _opt_ptr(tables), _opt_ptr(lens), C.byref(h)))
        self.handle = h.value
        ptrs = [C.c_void_p() for _ in range(3)]
        dev._L.tq_pages_data(C.c_void_p(self.handle), *(C.byref(p) for p in ptrs))
        self.refs, self.tables, self.lens = (Buffer(dev, p.value, n, _lib.I32, owns=False)
                                             for p, n in zip(ptrs, (n_pages, n_seqs * max_pages, n_seqs)))
        if arrays is not None:
            self.set_arrays(arrays)

    def set_arrays(self, arrays) -> None:
        arrays = list(arrays)
        row = arrays[0].nbytes // (self.n_pages * self.page_rows) if arrays else 0
        if any(a.nbytes != self.n_pages * self.page_rows * row for a in arrays):
            raise TangqError(TQ_EINVAL, "PagePool: every array holds n_pages * page_rows rows of one size")
        self._keep.append(arrays)
        bases = (C.c_void_p * len(arrays))(*[a.ptr for a in arrays])
        self.dev._check(self.dev._L.tq_pages_arrays(C.c_void_p(self.handle), bases, len(arrays), row))

    def _ints(self, v, n: int | None):
        """(Buffer, how many of its values count) of a Buffer or a sequence of ints."""
        if v is None:
            return None, n
        if not isinstance(v, Buffer):
            if self.dev.capturing:
                raise TangqError(TQ_EINVAL, "PagePool: a recorded call reads its lists when it is replayed: they have to be Buffers that live as long")
            v = self.dev.upload(np.asarray(v, np.int32), _lib.I32)
        if v.dtype != _lib.I32 or (n is not None and v.n < n):
            raise TangqError(TQ_EINVAL, f"PagePool: a list of {v.n} values where {n} of int32 are needed")
        return v, v.n if n is None else n

    def extend(self, seqs, n: int | None = None, counts=None) -> None:
        """Makes room for the next tokens (one, or `counts`) of each listed sequence and counts them to its length: new pages, and a
        copy of a partly filled last page that another sequence holds too."""
        seqs, n = self._ints(seqs, n)
        counts, _ = self._ints(counts, n)
        self.dev._check(self.dev._L.tq_pages_extend(C.c_void_p(self.handle), C.c_void_p(seqs.ptr), _opt_ptr(counts), n))

    def fork(self, src, dst, n: int | None = None, keep=None) -> None:
        """Sequence dst[i], empty so far, becomes what src[i] is (or its first keep[i] positions), in the same pages."""
        src, n = self._ints(src, n)
        dst, _ = self._ints(dst, n)
        keep, _ = self._ints(keep, n)
        self.dev._check(self.dev._L.tq_pages_fork(C.c_void_p(self.handle), C.c_void_p(src.ptr), C.c_void_p(dst.ptr), _opt_ptr(keep), n))

    def free(self, seqs, n: int | None = None) -> None:
        """The listed sequences give their pages back and are empty."""
        seqs, n = self._ints(seqs, n)
        self.dev._check(self.dev._L.tq_pages_free(C.c_void_p(self.handle), C.c_void_p(seqs.ptr), n))

    def compact(self, used: Buffer | None = None) -> None:
        """Moves the pages in use to the front of the pool; `used` receives how many there are."""
        if used is not None and (used.dtype != _lib.I32 or used.n < 1):
            raise TangqError(TQ_EINVAL, "PagePool: the number of pages in use needs an int32")
        self.dev._check(self.dev._L.tq_pages_compact(C.c_void_p(self.handle), _opt_ptr(used)))

    def state(self):
        """(refs [n_pages], tables [n_seqs, max_pages], lens [n_seqs]) as numpy arrays."""
        return self.refs.to_vec(), self.tables.to_vec().reshape(self.n_seqs, self.max_pages), self.lens.to_vec()

    def destroy(self) -> None:
        if self.handle:
            self.dev._L.tq_pages_destroy(C.c_void_p(self.handle))
            self.handle = 0

    def __del__(self):
        try:
            self.destroy()
        except Exception:
            pass
