"""The paged 4-bit key/value cache: block tables on the device, the cache
write and read, attention over it, and the choice of pages for sparse
attention (include/moe_hip.h, "the paged 4-bit key/value cache").

The reference keeps one f32 cache per sequence, reserved to the context's end
(State, src/model.rs:93-114, 732-733).  Here sequences take pages of positions
from a pool as they grow (PageTable), a layer's keys and values are held as
the reference's Q4 blocks (KvCache: 4.5 bits a value instead of 32), and a
row may attend to every position or to the pages it scores highest.

Every method queues its kernels on `stream` (torch's current stream of the
cache's device when None) and returns; nothing waits for the device, so a
whole decode step can be captured into a graph.  Arguments that do not fit
raise ValueError before anything is queued.
"""
from __future__ import annotations

import ctypes as C
import functools
from typing import Optional

from . import _lib as L

try:
    import torch
except ImportError:  # pragma: no cover - torch is part of the image
    torch = None


# A step of few rows is as long as its calls take to queue, so what a call has
# to check is checked in few steps, and the addresses of an object's own tensors
# are taken when it is made.


def _need(ok: bool, what: str) -> None:
    if not ok:
        raise ValueError(what)


def _fits(**numbers) -> None:
    """Numbers that the library takes in 32 bits: ctypes would drop the rest."""
    for name, n in numbers.items():
        if not -2 ** 31 <= n < 2 ** 31:
            raise ValueError(f"{name} {n}: a number of 32 bits")


def _refused(rc: int, what: str) -> None:
    """The error of a call that the library did not make."""
    try:
        L.check(rc, what)
    except L.MoeError as e:
        if e.code in (L.MOE_EINVAL, L.MOE_EUNSUP):
            raise ValueError(str(e)) from None
        raise


def _ids(t, dtype, n: int, name: str) -> None:
    if t.dtype != dtype or t.shape != (n,) or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous {str(dtype)[6:]} tensor of {n}")


def _rows(t, rows: int, cols: int, name: str) -> int:
    """The row stride of float32 [rows, cols] with contiguous rows."""
    if t.dtype != torch.float32 or t.shape != (rows, cols):
        raise ValueError(f"{name} must be float32 [{rows}, {cols}]")
    st = t.stride()
    if (st[1] != 1 and cols > 1) or (st[0] < cols and rows > 1):
        raise ValueError(f"{name} must have contiguous rows that do not overlap: strides {st}")
    return st[0]


class _Fixed:
    """An object whose tensors' addresses are taken when it is made: its
    attributes stay what they were.  (Their contents may change; memory that
    another tensor should take needs another object.)"""

    def __setattr__(self, name, value):
        if name in self.__dict__ and name[0] != "_":
            raise AttributeError(f"{type(self).__name__}.{name} is fixed: its address is taken when the object is made")
        object.__setattr__(self, name, value)


class _OnDevice(_Fixed):
    """Where a call's kernels and scratch go."""

    device: "torch.device"

    def _check_device(self, *tensors) -> None:
        index = self._index
        for t in tensors:
            if t.get_device() != index:
                raise ValueError(f"a tensor on {t.device}; this is on {self.device}")
        if index < 0:
            raise ValueError(f"tensors on {self.device}: the kernels run on the GPU")

    def _on(self, stream) -> int:
        """The call's stream handle: torch's current one of this object's
        device when None."""
        if stream is None:
            return torch._C._cuda_getCurrentRawStream(self._index)
        if type(stream) is int:
            return stream
        index = getattr(stream, "device_index", self._index)
        if index != self._index:
            raise ValueError(f"a stream of cuda:{index}; this is on {self.device}")
        return stream.cuda_stream

    def _scratch(self, n: int, sp: int):
        """n bytes that stream sp owns.  The caching allocator hands a freed
        block to later work of the stream it was allocated on: the call's own,
        whichever is current.  Inside a capture it comes from the graph's own
        pool."""
        if sp == torch._C._cuda_getCurrentRawStream(self._index):
            return torch.empty(n, dtype=torch.uint8, device=self.device)
        s = torch.cuda.ExternalStream(sp, device=self.device) if sp else torch.cuda.default_stream(self.device)
        with torch.cuda.stream(s):
            return torch.empty(n, dtype=torch.uint8, device=self.device)


def _on_its_device(call):
    """Run a method with its object's device current."""
    @functools.wraps(call)
    def run(self, *args, **kw):
        index = self._index
        if index < 0 or torch._C._cuda_getDevice() == index:
            return call(self, *args, **kw)
        with torch.cuda.device(index):
            return call(self, *args, **kw)
    return run


class Rows(_Fixed):
    """What PageTable.advance says of a step's rows: `row_start` int32
    [sequences + 1], `seq`, `pos` int32 and `slot` int64 [rows], `status` int32
    [sequences].  Their number of rows is what a step has room for."""

    def __init__(self, row_start, seq, pos, slot, status):
        n = seq.shape[0]
        _fits(rows=n, sequences=status.shape[0])
        _ids(seq, torch.int32, n, "seq")
        _ids(pos, torch.int32, n, "pos")
        _ids(slot, torch.int64, n, "slot")
        _ids(row_start, torch.int32, status.shape[0] + 1, "row_start")
        _ids(status, torch.int32, status.shape[0], "status")
        self.row_start, self.seq, self.pos, self.slot, self.status = row_start, seq, pos, slot, status
        self.device, self._index = seq.device, seq.get_device()
        _need(all(t.device == self.device for t in (pos, slot, row_start, status)), "rows on several devices")
        self._args = (n, row_start.data_ptr(), seq.data_ptr(), pos.data_ptr(), slot.data_ptr(), status.data_ptr())
        self.n_seq = status.shape[0]

    @staticmethod
    def new(n_seq: int, rows: int, device) -> "Rows":
        e = lambda n, t=torch.int32: torch.empty(n, dtype=t, device=device)  # noqa: E731
        return Rows(e(n_seq + 1), e(rows), e(rows), e(rows, torch.int64), e(n_seq))


class PageTable(_OnDevice):
    """Which pages each sequence holds: `table` int32 [sequences, pages],
    `length` int32 [sequences] positions, and the pool's free pages, `state` =
    (head, count) of the ring `ring` int32 [pages of the pool]."""

    def __init__(self, table, length, ring, state, page: int):
        _need(table.dtype == torch.int32 and table.dim() == 2 and table.is_contiguous(),
              "table must be a contiguous int32 [sequences, pages] tensor")
        _fits(page=page, sequences=table.shape[0], pages=table.shape[1], pool=ring.shape[0])
        _ids(length, torch.int32, table.shape[0], "length")
        _ids(ring, torch.int32, ring.shape[0], "ring")
        _ids(state, torch.int32, 2, "state")
        self.table, self.length, self.ring, self.state, self.page = table, length, ring, state, page
        self.device, self._index = table.device, table.get_device()
        _need(all(t.device == self.device for t in (length, ring, state)), "a table on several devices")
        self._where = (table.data_ptr(), table.shape[1], page, ring.data_ptr(), ring.shape[0])
        self._now = (length.data_ptr(), state.data_ptr())
        self._bytes = 0

    @staticmethod
    def new(n_seq: int, max_pages: int, n_pages: int, page: int, device) -> "PageTable":
        """Empty sequences, every page free."""
        return PageTable(torch.full((n_seq, max_pages), -1, dtype=torch.int32, device=device),
                         torch.zeros(n_seq, dtype=torch.int32, device=device),
                         torch.arange(n_pages, dtype=torch.int32, device=device),
                         torch.tensor([0, n_pages], dtype=torch.int32, device=device), page)

    @_on_its_device
    def advance(self, add, rows: Rows, out: Optional["PageTable"] = None, stream=None) -> Rows:
        """Give sequence i add[i] more positions (int32; below 0: end it and
        free its pages) and fill `rows` (moe_pages_advance).  The new lengths
        and state go to `out` (a PageTable over the same table and ring) or
        replace this one's."""
        out = self if out is None else out
        n = self.table.shape[0]
        _ids(add, torch.int32, n, "add")
        _need(rows.n_seq == n, f"rows of {rows.n_seq} sequences, the table has {n}")
        _need(out._where == self._where, "out has another table or ring")
        self._check_device(add, rows.seq)
        if not self._bytes:
            b = C.c_uint64()
            _refused(L.lib().moe_pages_workspace_size(n, C.byref(b)), "moe_pages_workspace_size")
            self._bytes = b.value
        sp = self._on(stream)
        ws = self._scratch(self._bytes, sp)
        rc = L.lib().moe_pages_advance(n, self._now[0], add.data_ptr(), out._now[0], *self._where, self._now[1],
                                       out._now[1], *rows._args, ws.data_ptr(), self._bytes, sp)
        if rc:
            _refused(rc, "moe_pages_advance")
        return rows


class KvCache(_OnDevice):
    """One layer's keys and values in 4 bits: `pool` uint8, pages found
    through `table` (a PageTable's).  With `means` (float16 [pages, kv heads,
    key width]) full pages keep the mean key that select() scores them by."""

    def __init__(self, pool, table, *, n_kv: int, qd: int, vd: int, page: int, means=None):
        _need(pool.dtype == torch.uint8 and pool.dim() == 1 and pool.is_contiguous(),
              "pool must be a contiguous one-dimensional uint8 tensor")
        _need(table.dtype == torch.int32 and table.dim() == 2 and table.is_contiguous(),
              "table must be a contiguous int32 [sequences, pages] tensor")
        n_pages = pool.shape[0] // self.page_bytes(n_kv, qd, vd, page)
        _need(n_pages >= 1, f"a pool of {pool.shape[0]} bytes holds no page")
        _fits(sequences=table.shape[0], pages=table.shape[1], pool=n_pages)
        if means is not None:
            _need(means.dtype == torch.float16 and means.is_contiguous() and tuple(means.shape) == (n_pages, n_kv, qd),
                  f"means must be a contiguous float16 [{n_pages}, {n_kv}, {qd}] tensor")
        self.pool, self.table, self.means = pool, table, means
        self.n_kv, self.qd, self.vd, self.page, self.n_pages = n_kv, qd, vd, page, n_pages
        self.device, self._index = pool.device, pool.get_device()
        _need(table.device == pool.device and (means is None or means.device == pool.device),
              "a cache on several devices")
        self.c = L.Kv4C(pool=pool.data_ptr(), pool_bytes=pool.shape[0], table=table.data_ptr(),
                        means=None if means is None else means.data_ptr(), n_seq=table.shape[0],
                        max_pages=table.shape[1], n_pages=n_pages, page=page, n_kv=n_kv, qd=qd, vd=vd)
        self._c = C.byref(self.c)
        self._positions = table.shape[1] * page
        self._sizes = {}

    @staticmethod
    def page_bytes(n_kv: int, qd: int, vd: int, page: int) -> int:
        """Bytes of a page; ValueError for sizes the cache does not hold."""
        _fits(page=page, n_kv=n_kv, qd=qd, vd=vd)
        one = L.Kv4C(n_pages=1, page=page, n_kv=n_kv, qd=qd, vd=vd)
        b = C.c_uint64()
        _refused(L.lib().moe_kv4_pool_size(C.byref(one), C.byref(b)), "moe_kv4_pool_size")
        return b.value

    @staticmethod
    def new(n_pages: int, table, *, n_kv: int, qd: int, vd: int, page: int, means: bool = False) -> "KvCache":
        dev = table.device
        pool = torch.zeros(n_pages * KvCache.page_bytes(n_kv, qd, vd, page), dtype=torch.uint8, device=dev)
        m = torch.zeros((n_pages, n_kv, qd), dtype=torch.float16, device=dev) if means else None
        return KvCache(pool, table, n_kv=n_kv, qd=qd, vd=vd, page=page, means=m)

    def _size(self, name: str, *args) -> int:
        n = self._sizes.get((name, args))
        if n is None:
            b = C.c_uint64()
            _refused(getattr(L.lib(), name)(self._c, *args, C.byref(b)), name)
            if len(self._sizes) > 256:
                self._sizes.clear()
            n = self._sizes[name, args] = b.value
        return n

    @_on_its_device
    def store(self, k, v, slots, stream=None) -> None:
        """Write rows k [rows, kv heads * key width], v [rows, kv heads *
        value width] (float32) into `slots` (int64, distinct; rows of negative
        slots are skipped)."""
        n = k.shape[0]
        _fits(rows=n)
        ks, vs = _rows(k, n, self.n_kv * self.qd, "k"), _rows(v, n, self.n_kv * self.vd, "v")
        _ids(slots, torch.int64, n, "slots")
        self._check_device(k, v, slots)
        rc = L.lib().moe_kv4_store(self._c, k.data_ptr(), ks, v.data_ptr(), vs, n, slots.data_ptr(), self._on(stream))
        if rc:
            _refused(rc, "moe_kv4_store")

    @_on_its_device
    def load(self, slots, k=None, v=None, stream=None) -> None:
        """Read the rows of `slots` into k and v (float32, either may be
        None); rows of negative slots are left as they were."""
        n = slots.shape[0]
        _fits(rows=n)
        _ids(slots, torch.int64, n, "slots")
        ks = 0 if k is None else _rows(k, n, self.n_kv * self.qd, "k")
        vs = 0 if v is None else _rows(v, n, self.n_kv * self.vd, "v")
        self._check_device(slots, *(t for t in (k, v) if t is not None))
        rc = L.lib().moe_kv4_load(self._c, slots.data_ptr(), n, None if k is None else k.data_ptr(), ks,
                                  None if v is None else v.data_ptr(), vs, self._on(stream))
        if rc:
            _refused(rc, "moe_kv4_load")

    def _query(self, q, seq, pos, max_pos):
        """(rows, heads, row stride) of a call's queries."""
        if not 0 <= max_pos < self._positions:
            raise ValueError(f"max_pos {max_pos}: the table has {self._positions} positions a sequence")
        n, width = q.shape if q.dim() == 2 else (-1, 0)
        heads = width // self.qd
        if heads < 1 or heads % self.n_kv:
            raise ValueError(f"queries of {tuple(q.shape)}: rows of a multiple of {self.n_kv} heads of {self.qd}")
        qs = _rows(q, n, heads * self.qd, "q")
        _ids(seq, torch.int32, n, "seq")
        _ids(pos, torch.int32, n, "pos")
        return n, heads, qs

    def _lists(self, t, n: int, name: str) -> int:
        if t.dtype != torch.int32 or t.dim() != 3 or t.shape[:2] != (n, self.n_kv) or t.shape[2] < 1 or \
                not t.is_contiguous():
            raise ValueError(f"{name} must be a contiguous int32 [{n}, {self.n_kv}, pages] tensor")
        return t.shape[2]

    @_on_its_device
    def attend(self, q, seq, pos, out, *, max_pos: int, scale: float, window: int = 0, pages=None, stream=None) -> None:
        """Causal attention of rows q [rows, heads * key width] into out
        [rows, heads * value width] (moe_kv4_attention): row r of sequence
        seq[r] at position pos[r] (-1: left as it was), no position above
        max_pos (a loose bound changes nothing but the time: runs are split as
        if they went that far, 4 sequences at 300 positions 10 us with their own
        bound, 31 with one of 65535), over the last `window` positions when that is above 0, over
        the pages `pages` lists (select's int32 [rows, kv heads, n]) when
        given."""
        n, heads, qs = self._query(q, seq, pos, max_pos)
        if not -2 ** 31 <= window < 2 ** 31:
            _fits(window=window)
        os = _rows(out, n, heads * self.vd, "out")
        if pages is None:
            n_sel, lists = 0, None
            self._check_device(q, seq, pos, out)
        else:
            n_sel, lists = self._lists(pages, n, "pages"), pages.data_ptr()
            self._check_device(q, seq, pos, out, pages)
        need = self._size("moe_kv4_attention_workspace_size", n, heads, max_pos, window, n_sel)
        sp = self._on(stream)
        ws = self._scratch(need, sp) if need else None
        rc = L.lib().moe_kv4_attention(self._c, q.data_ptr(), qs, n, heads, scale, seq.data_ptr(), pos.data_ptr(), max_pos,
                                       window, lists, n_sel, out.data_ptr(), os, ws.data_ptr() if need else None, need, sp)
        if rc:
            _refused(rc, "moe_kv4_attention")

    @_on_its_device
    def select(self, q, seq, pos, lists, *, max_pos: int, sinks: int = 1, recent: int = 1, stream=None):
        """Fill lists (int32 [rows, kv heads, n]) with the n pages each row
        and kv head reads (moe_kv4_select): the first `sinks`, the last
        `recent`, then by score; -1 behind the last."""
        if self.means is None:
            raise ValueError("the cache keeps no mean keys")
        n, heads, qs = self._query(q, seq, pos, max_pos)
        n_sel = self._lists(lists, n, "lists")
        if sinks < 0 or recent < 1 or sinks + recent > n_sel:
            raise ValueError(f"{sinks} first and {recent} last pages of {n_sel}")
        self._check_device(q, seq, pos, lists)
        need = self._size("moe_kv4_select_workspace_size", n, max_pos)
        sp = self._on(stream)
        ws = self._scratch(need, sp) if need else None
        rc = L.lib().moe_kv4_select(self._c, q.data_ptr(), qs, n, heads, seq.data_ptr(), pos.data_ptr(), max_pos, sinks,
                                    recent, n_sel, lists.data_ptr(), ws.data_ptr() if need else None, need, sp)
        if rc:
            _refused(rc, "moe_kv4_select")
        return lists
