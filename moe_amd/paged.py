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
from typing import Optional

from . import _lib as L

try:
    import torch
except ImportError:  # pragma: no cover - torch is part of the image
    torch = None


def _need(ok: bool, what: str) -> None:
    if not ok:
        raise ValueError(what)


def _ids(t, dtype, n: int, name: str) -> None:
    _need(t.dtype == dtype and t.dim() == 1 and t.is_contiguous() and t.shape[0] == n,
          f"{name} must be a contiguous {str(dtype)[6:]} tensor of {n}")


def _rows(t, rows: int, cols: int, name: str) -> None:
    _need(t.dtype == torch.float32 and t.dim() == 2 and t.shape[0] == rows and t.shape[1] == cols
          and (cols == 1 or t.stride(1) == 1) and (rows <= 1 or t.stride(0) >= 0),
          f"{name} must be float32 [{rows}, {cols}] with contiguous rows")


class _OnDevice:
    """Where a call's kernels and scratch go."""

    device: "torch.device"

    def _call(self, tensors, run, stream):
        """run(stream handle, scratch) on this object's device; scratch(n)
        gives n bytes that the call's stream owns."""
        dev = self.device
        for t in tensors:
            if t is not None and t.device != dev:
                raise ValueError(f"a tensor on {t.device}; the cache is on {dev}")
        if dev.type != "cuda":
            raise ValueError(f"a cache on {dev}: the kernels run on the GPU")
        if torch.cuda.current_device() != dev.index:
            with torch.cuda.device(dev):
                return self._call(tensors, run, stream)
        mine = torch.cuda.current_stream().cuda_stream
        sp = mine if stream is None else stream if type(stream) is int else stream.cuda_stream

        def scratch(n: int):
            # The caching allocator hands a freed block to later work of the
            # stream it was allocated on: the call's own, whichever is current.
            # Inside a capture it comes from the graph's own pool.
            if sp == mine:
                return torch.empty(n, dtype=torch.uint8, device=dev)
            s = torch.cuda.ExternalStream(sp, device=dev) if sp else torch.cuda.default_stream(dev)
            with torch.cuda.stream(s):
                return torch.empty(n, dtype=torch.uint8, device=dev)

        return run(sp, scratch)


class Rows:
    """What PageTable.advance says of a step's rows: `row_start` int32
    [sequences + 1], `seq`, `pos` int32 and `slot` int64 [rows], `status` int32
    [sequences].  Their number of rows is what a step has room for."""

    def __init__(self, row_start, seq, pos, slot, status):
        n = seq.shape[0]
        _ids(seq, torch.int32, n, "seq")
        _ids(pos, torch.int32, n, "pos")
        _ids(slot, torch.int64, n, "slot")
        _ids(row_start, torch.int32, status.shape[0] + 1, "row_start")
        _ids(status, torch.int32, status.shape[0], "status")
        self.row_start, self.seq, self.pos, self.slot, self.status = row_start, seq, pos, slot, status

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
        _ids(length, torch.int32, table.shape[0], "length")
        _ids(ring, torch.int32, ring.shape[0], "ring")
        _ids(state, torch.int32, 2, "state")
        self.table, self.length, self.ring, self.state, self.page = table, length, ring, state, page
        self.device = table.device
        self._scratch = 0

    @staticmethod
    def new(n_seq: int, max_pages: int, n_pages: int, page: int, device) -> "PageTable":
        """Empty sequences, every page free."""
        return PageTable(torch.full((n_seq, max_pages), -1, dtype=torch.int32, device=device),
                         torch.zeros(n_seq, dtype=torch.int32, device=device),
                         torch.arange(n_pages, dtype=torch.int32, device=device),
                         torch.tensor([0, n_pages], dtype=torch.int32, device=device), page)

    def advance(self, add, rows: Rows, out: Optional["PageTable"] = None, stream=None) -> Rows:
        """Give sequence i add[i] more positions (int32; below 0: end it and
        free its pages) and fill `rows` (moe_pages_advance).  The new lengths
        and state go to `out` (a PageTable over the same table and ring) or
        replace this one's."""
        out = self if out is None else out
        n = self.table.shape[0]
        _ids(add, torch.int32, n, "add")
        _need(rows.status.shape[0] == n, f"rows of {rows.status.shape[0]} sequences, the table has {n}")
        _need(out is self or (out.table.data_ptr() == self.table.data_ptr() and out.page == self.page
                              and out.table.shape == self.table.shape and out.ring.shape == self.ring.shape
                              and out.ring.data_ptr() == self.ring.data_ptr()), "out has another table or ring")
        if not self._scratch:
            b = C.c_uint64()
            L.check(L.lib().moe_pages_workspace_size(n, C.byref(b)), "moe_pages_workspace_size")
            self._scratch = b.value

        def run(sp, scratch):
            ws = scratch(self._scratch)
            rc = L.lib().moe_pages_advance(
                n, self.length.data_ptr(), add.data_ptr(), out.length.data_ptr(), self.table.data_ptr(),
                self.table.shape[1], self.page, self.ring.data_ptr(), self.ring.shape[0], self.state.data_ptr(),
                out.state.data_ptr(), rows.seq.shape[0], rows.row_start.data_ptr(), rows.seq.data_ptr(),
                rows.pos.data_ptr(), rows.slot.data_ptr(), rows.status.data_ptr(), ws.data_ptr(), self._scratch, sp)
            if rc:
                L.check(rc, "moe_pages_advance")

        self._call((add, rows.seq, rows.pos, rows.slot, rows.row_start, rows.status, self.length, self.ring, self.state,
                    out.length, out.state), run, stream)
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
        if means is not None:
            _need(means.dtype == torch.float16 and means.is_contiguous() and tuple(means.shape) == (n_pages, n_kv, qd),
                  f"means must be a contiguous float16 [{n_pages}, {n_kv}, {qd}] tensor")
        self.pool, self.table, self.means = pool, table, means
        self.n_kv, self.qd, self.vd, self.page, self.n_pages = n_kv, qd, vd, page, n_pages
        self.device = pool.device
        self.c = L.Kv4C(pool=pool.data_ptr(), pool_bytes=pool.shape[0], table=table.data_ptr(),
                        means=None if means is None else means.data_ptr(), n_seq=table.shape[0],
                        max_pages=table.shape[1], n_pages=n_pages, page=page, n_kv=n_kv, qd=qd, vd=vd)
        self._c = C.byref(self.c)
        self._sizes = {}

    @staticmethod
    def page_bytes(n_kv: int, qd: int, vd: int, page: int) -> int:
        """Bytes of a page; ValueError for sizes the cache does not hold."""
        one = L.Kv4C(n_pages=1, page=page, n_kv=n_kv, qd=qd, vd=vd)
        b = C.c_uint64()
        try:
            L.check(L.lib().moe_kv4_pool_size(C.byref(one), C.byref(b)), "moe_kv4_pool_size")
        except L.MoeError as e:
            raise ValueError(str(e)) from None
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
            L.check(getattr(L.lib(), name)(self._c, *args, C.byref(b)), name)
            if len(self._sizes) > 256:
                self._sizes.clear()
            n = self._sizes[name, args] = b.value
        return n

    def store(self, k, v, slots, stream=None) -> None:
        """Write rows k [rows, kv heads * key width], v [rows, kv heads *
        value width] (float32) into `slots` (int64, distinct; rows of negative
        slots are skipped)."""
        n = k.shape[0]
        _rows(k, n, self.n_kv * self.qd, "k")
        _rows(v, n, self.n_kv * self.vd, "v")
        _ids(slots, torch.int64, n, "slots")

        def run(sp, scratch):
            rc = L.lib().moe_kv4_store(self._c, k.data_ptr(), k.stride(0), v.data_ptr(), v.stride(0), n,
                                       slots.data_ptr(), sp)
            if rc:
                L.check(rc, "moe_kv4_store")

        self._call((k, v, slots, self.table, self.means), run, stream)

    def load(self, slots, k=None, v=None, stream=None) -> None:
        """Read the rows of `slots` into k and v (float32, either may be
        None); rows of negative slots are left as they were."""
        n = slots.shape[0]
        _ids(slots, torch.int64, n, "slots")
        if k is not None:
            _rows(k, n, self.n_kv * self.qd, "k")
        if v is not None:
            _rows(v, n, self.n_kv * self.vd, "v")

        def run(sp, scratch):
            rc = L.lib().moe_kv4_load(self._c, slots.data_ptr(), n, None if k is None else k.data_ptr(),
                                      0 if k is None else k.stride(0), None if v is None else v.data_ptr(),
                                      0 if v is None else v.stride(0), sp)
            if rc:
                L.check(rc, "moe_kv4_load")

        self._call((slots, k, v, self.table), run, stream)

    def _query(self, q, seq, pos) -> int:
        n = q.shape[0]
        heads = q.shape[1] // self.qd
        _need(heads >= 1 and heads % self.n_kv == 0, f"queries of {q.shape[1]} values: not a multiple of {self.n_kv} kv "
              f"heads of {self.qd}")
        _rows(q, n, heads * self.qd, "q")
        _ids(seq, torch.int32, n, "seq")
        _ids(pos, torch.int32, n, "pos")
        return heads

    def attend(self, q, seq, pos, out, *, max_pos: int, scale: float, window: int = 0, pages=None, stream=None) -> None:
        """Causal attention of rows q [rows, heads * key width] into out
        [rows, heads * value width] (moe_kv4_attention): row r of sequence
        seq[r] at position pos[r] (-1: left as it was), no position above
        max_pos, over the last `window` positions when that is above 0, over
        the pages `pages` lists (select's int32 [rows, kv heads, n]) when
        given."""
        heads = self._query(q, seq, pos)
        n = q.shape[0]
        _rows(out, n, heads * self.vd, "out")
        n_sel = 0
        if pages is not None:
            _need(pages.dtype == torch.int32 and pages.dim() == 3 and pages.is_contiguous()
                  and pages.shape[0] == n and pages.shape[1] == self.n_kv and pages.shape[2] >= 1,
                  f"pages must be a contiguous int32 [{n}, {self.n_kv}, pages] tensor")
            n_sel = pages.shape[2]
        need = self._size("moe_kv4_attention_workspace_size", n, heads, max_pos, window, n_sel)

        def run(sp, scratch):
            ws = scratch(need) if need else None
            rc = L.lib().moe_kv4_attention(self._c, q.data_ptr(), q.stride(0), n, heads, scale, seq.data_ptr(),
                                           pos.data_ptr(), max_pos, window, None if pages is None else pages.data_ptr(),
                                           n_sel, out.data_ptr(), out.stride(0), None if ws is None else ws.data_ptr(),
                                           need, sp)
            if rc:
                L.check(rc, "moe_kv4_attention")

        self._call((q, seq, pos, out, pages, self.table), run, stream)

    def select(self, q, seq, pos, lists, *, max_pos: int, sinks: int = 1, recent: int = 1, stream=None):
        """Fill lists (int32 [rows, kv heads, n]) with the n pages each row
        and kv head reads (moe_kv4_select): the first `sinks`, the last
        `recent`, then by score; -1 behind the last."""
        _need(self.means is not None, "the cache keeps no mean keys")
        heads = self._query(q, seq, pos)
        n = q.shape[0]
        _need(lists.dtype == torch.int32 and lists.dim() == 3 and lists.is_contiguous()
              and lists.shape[0] == n and lists.shape[1] == self.n_kv and lists.shape[2] >= 1,
              f"lists must be a contiguous int32 [{n}, {self.n_kv}, pages] tensor")
        _need(sinks >= 0 and recent >= 1 and sinks + recent <= lists.shape[2],
              f"{sinks} first and {recent} last pages of {lists.shape[2]}")
        need = self._size("moe_kv4_select_workspace_size", n, max_pos)

        def run(sp, scratch):
            ws = scratch(max(need, 16))
            rc = L.lib().moe_kv4_select(self._c, q.data_ptr(), q.stride(0), n, heads, seq.data_ptr(), pos.data_ptr(),
                                        max_pos, sinks, recent, lists.shape[2], lists.data_ptr(), ws.data_ptr(), need,
                                        sp)
            if rc:
                L.check(rc, "moe_kv4_select")

        self._call((q, seq, pos, lists, self.table, self.means), run, stream)
        return lists
