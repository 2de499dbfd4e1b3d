"""The paged cache's entry points on the CPU: what they refuse, before
anything is queued, and the layout's sizes."""
import ctypes as C

import pytest
import torch

from moe_amd import _lib as L
from moe_amd.paged import KvCache, PageTable, Rows

P = 0x10000  # an address that no refused call reads


@pytest.fixture(scope="module")
def lib():
    if not L.LIB_PATH.exists():
        from moe_amd.build import build

        build()
    return L.lib()


def kv4(**kw):
    c = dict(pool=P, pool_bytes=1 << 40, table=P, means=P, n_seq=4, max_pages=10, n_pages=100, page=64, n_kv=2, qd=64, vd=64)
    c.update(kw)
    return L.Kv4C(**c)


BAD_CACHES = [dict(pool=None), dict(table=None), dict(pool=P + 8), dict(means=P + 2), dict(pool_bytes=100 * 2 * 2 * 2304 - 1),
              dict(n_seq=0), dict(max_pages=0), dict(n_pages=0), dict(n_kv=0), dict(page=16), dict(page=48), dict(page=8192),
              dict(page=0), dict(page=4096, max_pages=1 << 20), dict(qd=0), dict(qd=48), dict(vd=288), dict(vd=-32),
              dict(n_pages=2 ** 31 - 1, page=4096, n_kv=2 ** 31 - 1)]


def attention(lib, c, q=P, stride=512, rows=3, heads=8, seq=P, pos=P, max_pos=100, window=0, lists=None, n_sel=0, out=P,
              ws=P, ws_bytes=1 << 40):
    return lib.moe_kv4_attention(C.byref(c), q, stride, rows, heads, 0.125, seq, pos, max_pos, window, lists, n_sel, out,
                                 stride, ws, ws_bytes, None)


def select(lib, c, q=P, rows=3, heads=8, seq=P, pos=P, max_pos=100, sinks=1, recent=1, n_sel=4, lists=P, ws=P, ws_bytes=1 << 30):
    return lib.moe_kv4_select(C.byref(c), q, 512, rows, heads, seq, pos, max_pos, sinks, recent, n_sel, lists, ws, ws_bytes,
                              None)


def store(lib, c, k=P, v=P, rows=3, slots=P):
    return lib.moe_kv4_store(C.byref(c), k, 128, v, 128, rows, slots, None)


def load(lib, c, slots=P, rows=3):
    return lib.moe_kv4_load(C.byref(c), slots, rows, P, 128, P, 128, None)


@pytest.mark.parametrize("call", [attention, select, store, load])
@pytest.mark.parametrize("bad", BAD_CACHES, ids=str)
def test_refuses_bad_caches(lib, call, bad):
    assert call(lib, kv4(**bad)) in (L.MOE_EINVAL, L.MOE_EUNSUP)
    assert lib.moe_last_error()


@pytest.mark.parametrize("call", [attention, select, store, load])
def test_no_rows_are_no_work(lib, call):
    """Null pointers and all: torch's empty tensors have no address."""
    kw = {attention: dict(q=None, seq=None, pos=None, out=None), select: dict(q=None, seq=None, pos=None, lists=None),
          store: dict(k=None, v=None, slots=None), load: dict(slots=None)}[call]
    assert call(lib, kv4(), rows=0, **kw) == L.MOE_OK
    assert call(lib, kv4(), rows=-1) == L.MOE_EINVAL
    for k in kw:
        assert call(lib, kv4(), **{k: None}) == L.MOE_EINVAL


LONG = dict(max_pages=2000, max_pos=100000)  # positions that go to several blocks


@pytest.mark.parametrize("bad", [dict(heads=7), dict(heads=0), dict(heads=-2), dict(max_pos=-1), dict(max_pos=640),
                                 dict(lists=P, n_sel=0), dict(lists=P, n_sel=-1), dict(ws=None, **LONG),
                                 dict(ws=P + 8, **LONG), dict(ws_bytes=1000, **LONG)], ids=str)
def test_attention_refuses(lib, bad):
    bad = dict(bad)
    assert attention(lib, kv4(max_pages=bad.pop("max_pages", 10)), **bad) == L.MOE_EINVAL


MANY = dict(max_pages=9000, max_pos=64 * 8000)  # pages whose scores go through the workspace


@pytest.mark.parametrize("bad", [dict(heads=7), dict(max_pos=-1), dict(max_pos=640), dict(sinks=-1), dict(recent=0),
                                 dict(sinks=3, recent=2), dict(sinks=2 ** 31 - 1, recent=2 ** 31 - 1), dict(n_sel=0),
                                 dict(ws=None, **MANY), dict(ws=P + 8, **MANY), dict(ws_bytes=16, **MANY)], ids=str)
def test_select_refuses(lib, bad):
    bad = dict(bad)
    assert select(lib, kv4(max_pages=bad.pop("max_pages", 10)), **bad) == L.MOE_EINVAL


def test_select_needs_means(lib):
    assert select(lib, kv4(means=None)) == L.MOE_EINVAL


def advance(lib, n=4, length=P, add=P, length_out=P, table=P, max_pages=10, page=64, ring=P, n_pages=100, state=P, state_out=P,
            rows=5, row_start=P, seq=P, pos=P, slot=P, status=P, ws=P, ws_bytes=1 << 20):
    return lib.moe_pages_advance(n, length, add, length_out, table, max_pages, page, ring, n_pages, state, state_out, rows,
                                 row_start, seq, pos, slot, status, ws, ws_bytes, None)


@pytest.mark.parametrize("bad", [dict(n=0), dict(n=-1), dict(max_pages=0), dict(n_pages=0), dict(rows=-1), dict(page=31),
                                 dict(page=96), dict(page=4096, max_pages=1 << 19), dict(ws=None), dict(ws=P + 4),
                                 dict(ws_bytes=15)] +
                         [{k: None} for k in ("length", "add", "length_out", "table", "ring", "state", "state_out",
                                              "row_start", "seq", "pos", "slot", "status")], ids=str)
def test_advance_refuses(lib, bad):
    assert advance(lib, **bad) == L.MOE_EINVAL


@pytest.mark.parametrize("qd,vd,page,n_kv", [(64, 64, 32, 1), (192, 128, 64, 16), (96, 32, 4096, 3), (256, 256, 128, 8)])
def test_page_bytes(lib, qd, vd, page, n_kv):
    assert KvCache.page_bytes(n_kv, qd, vd, page) == page * n_kv * (qd + vd) * 18 // 32


@pytest.mark.parametrize("bad", [(1, 64, 64, 33), (1, 40, 64, 32), (0, 64, 64, 32), (1, 64, 512, 32)], ids=str)
def test_page_bytes_refuses(lib, bad):
    with pytest.raises(ValueError):
        KvCache.page_bytes(*bad)


def cpu_cache(means=True):
    table = torch.zeros((3, 4), dtype=torch.int32)
    return KvCache.new(12, table, n_kv=2, qd=64, vd=32, page=32, means=means)


def ok_args():
    f = torch.zeros
    return dict(q=f(5, 256), seq=f(5, dtype=torch.int32), pos=f(5, dtype=torch.int32), out=f(5, 128),
                lists=f((5, 2, 3), dtype=torch.int32), k=f(5, 128), v=f(5, 64), slots=f(5, dtype=torch.int64))


def calls(c, a):
    return dict(attend=lambda: c.attend(a["q"], a["seq"], a["pos"], a["out"], max_pos=7, scale=1.0, pages=a["lists"]),
                select=lambda: c.select(a["q"], a["seq"], a["pos"], a["lists"], max_pos=7),
                store=lambda: c.store(a["k"], a["v"], a["slots"]),
                load=lambda: c.load(a["slots"], a["k"], a["v"]))


WRONG = {
    "q": [torch.zeros(5, 250), torch.zeros(5, 64), torch.zeros(5, 256).half(), torch.zeros(5, 512)[:, ::2], torch.zeros(4, 256)],
    "seq": [torch.zeros(5, dtype=torch.int64), torch.zeros(4, dtype=torch.int32), torch.zeros(10, dtype=torch.int32)[::2]],
    "pos": [torch.zeros(5), torch.zeros((5, 1), dtype=torch.int32)],
    "out": [torch.zeros(5, 256), torch.zeros(4, 128), torch.zeros(5, 128).double(), torch.zeros(128, 5).T],
    "lists": [torch.zeros((5, 1, 3), dtype=torch.int32), torch.zeros((5, 2, 3)), torch.zeros((5, 2, 0), dtype=torch.int32),
              torch.zeros((5, 2, 6), dtype=torch.int32)[..., ::2]],
    "k": [torch.zeros(5, 64), torch.zeros(5, 256)[:, ::2], torch.zeros(5, 128).bfloat16()],
    "v": [torch.zeros(5, 128), torch.zeros(4, 64)],
    "slots": [torch.zeros(5, dtype=torch.int32), torch.zeros(6, dtype=torch.int64)],
}
USES = {"attend": ("q", "seq", "pos", "out", "lists"), "select": ("q", "seq", "pos", "lists"), "store": ("k", "v", "slots"),
        "load": ("k", "v", "slots")}


@pytest.mark.parametrize("call", list(USES))
def test_wrong_tensors(lib, call):
    for name in USES[call]:
        for t in WRONG[name]:
            a = ok_args()
            a[name] = t
            with pytest.raises(ValueError):
                calls(cpu_cache(), a)[call]()
    # everything right but for the device
    with pytest.raises(ValueError, match="GPU"):
        calls(cpu_cache(), ok_args())[call]()


def test_select_without_means(lib):
    a = ok_args()
    with pytest.raises(ValueError, match="mean"):
        calls(cpu_cache(False), a)["select"]()
    with pytest.raises(ValueError):
        cpu_cache().select(a["q"], a["seq"], a["pos"], a["lists"], max_pos=7, sinks=2, recent=2)


def test_wrong_caches(lib):
    table, pool = torch.zeros((3, 4), dtype=torch.int32), torch.zeros(1 << 16, dtype=torch.uint8)
    ok = dict(n_kv=2, qd=64, vd=32, page=32)
    for p, t, kw in [(pool[:100], table, {}), (pool.view(2, -1), table, {}), (pool.view(torch.int8), table, {}),
                     (pool, table.long(), {}), (pool, table[:, ::2], {}), (pool, table, dict(qd=33)),
                     (pool, table, dict(means=torch.zeros((3, 2, 64)))),
                     (pool, table, dict(means=torch.zeros((3, 2, 64), dtype=torch.float16)))]:
        with pytest.raises(ValueError):
            KvCache(p, t, **{**ok, **kw})


def test_wrong_tables(lib):
    i = lambda *s: torch.zeros(s, dtype=torch.int32)  # noqa: E731
    with pytest.raises(ValueError):
        PageTable(i(3, 4), i(4), i(9), i(2), 32)
    with pytest.raises(ValueError):
        PageTable(i(3, 4), i(3), i(9), i(3), 32)
    with pytest.raises(ValueError):
        Rows(i(3), i(5), i(5), i(5), i(2))
    pt, other = PageTable(i(3, 4), i(3), i(9), i(2), 32), PageTable(i(3, 4), i(3), i(9), i(2), 32)
    for add, rows, out in [(i(4), Rows.new(3, 5, "cpu"), None), (i(3), Rows.new(2, 5, "cpu"), None),
                           (i(3), Rows.new(3, 5, "cpu"), other), (i(3).long(), Rows.new(3, 5, "cpu"), None)]:
        with pytest.raises(ValueError):
            pt.advance(add, rows, out=out)
    with pytest.raises(ValueError, match="GPU"):
        pt.advance(i(3), Rows.new(3, 5, "cpu"))


BIG = 2 ** 31 - 1


def test_refuses_what_no_launch_holds(lib):
    """Sizes whose blocks are more than a launch's: refused, nothing queued."""
    one = dict(n_kv=1, qd=32, vd=32, page=32, pool_bytes=1 << 60)
    for rows in (2 ** 24 - 255, BIG):
        assert store(lib, kv4(**one), rows=rows) == L.MOE_EUNSUP
        assert load(lib, kv4(**one), rows=rows) == L.MOE_EUNSUP
    assert attention(lib, kv4(**one), rows=BIG, heads=16) == L.MOE_EUNSUP
    assert attention(lib, kv4(**one), rows=2 ** 24, heads=16, lists=P, n_sel=1) == L.MOE_EUNSUP
    assert select(lib, kv4(**one), rows=2 ** 23, heads=1, ws_bytes=1 << 62) == L.MOE_EUNSUP
    for call in (attention, select, store, load):
        assert call(lib, kv4(n_kv=65536, pool_bytes=1 << 60)) != L.MOE_OK
    long = dict(one, max_pages=2 ** 26 - 1)
    assert select(lib, kv4(**long), rows=1, heads=1, max_pos=2 ** 31 - 33, ws_bytes=1 << 62) == L.MOE_EUNSUP


def test_refuses_lists_of_too_many_pages(lib):
    """More pages than positions have numbers."""
    n = C.c_uint64()
    for n_sel in (2 ** 25, BIG):
        assert attention(lib, kv4(), lists=P, n_sel=n_sel) == L.MOE_EINVAL
        assert select(lib, kv4(), n_sel=n_sel) == L.MOE_EINVAL
        assert lib.moe_kv4_attention_workspace_size(C.byref(kv4()), 3, 8, 100, 0, n_sel, C.byref(n)) == L.MOE_EINVAL


@pytest.mark.parametrize("bad", [dict(n=2 ** 24 + 1), dict(n=BIG), dict(n_pages=2 ** 30 + 1), dict(rows=2 ** 30), dict(rows=BIG)],
                         ids=str)
def test_advance_refuses_sizes_past_its_sums(lib, bad):
    assert advance(lib, ws_bytes=1 << 40, **bad) == L.MOE_EINVAL


@pytest.mark.parametrize("bad", [dict(max_pos=-1), dict(max_pos=128), dict(max_pos=2 ** 32 + 5), dict(max_pos=-2 ** 32 + 7)], ids=str)
def test_positions_past_the_table(lib, bad):
    """Refused as they are, not as what 32 bits hold of them."""
    c, a = cpu_cache(), ok_args()
    for call in (lambda **kw: c.attend(a["q"], a["seq"], a["pos"], a["out"], scale=1.0, **kw),
                 lambda **kw: c.select(a["q"], a["seq"], a["pos"], a["lists"], **kw)):
        with pytest.raises(ValueError, match="max_pos"):
            call(**bad)
        with pytest.raises(ValueError, match="GPU"):
            call(max_pos=127)


@pytest.mark.parametrize("window", [2 ** 31, 2 ** 32 + 16, -2 ** 31 - 1])
def test_windows_past_32_bits(lib, window):
    c, a = cpu_cache(), ok_args()
    with pytest.raises(ValueError, match="window"):
        c.attend(a["q"], a["seq"], a["pos"], a["out"], max_pos=7, scale=1.0, window=window)
    with pytest.raises(ValueError, match="GPU"):
        c.attend(a["q"], a["seq"], a["pos"], a["out"], max_pos=7, scale=1.0, window=2 ** 31 - 1)


def test_sizes_past_32_bits(lib):
    for bad in (dict(page=2 ** 32 + 32), dict(n_kv=2 ** 32 + 2), dict(qd=2 ** 32 + 64), dict(vd=-2 ** 32 + 64)):
        with pytest.raises(ValueError):
            KvCache.page_bytes(**{**dict(n_kv=2, qd=64, vd=32, page=32), **bad})
    i = lambda *s: torch.zeros(s, dtype=torch.int32)  # noqa: E731
    with pytest.raises(ValueError, match="page"):
        PageTable(i(3, 4), i(3), i(9), i(2), 2 ** 32 + 32)


def test_what_the_library_refuses_is_a_value_error(lib, monkeypatch):
    """Too many rows, pages of an odd size ...: as the module promises; a
    failure of the device stays what it is."""
    from moe_amd import paged

    with pytest.raises(ValueError):
        cpu_cache()._size("moe_kv4_attention_workspace_size", 3, 7, 10, 0, 0)
    monkeypatch.setattr(paged._OnDevice, "_check_device", lambda self, *t: None)
    monkeypatch.setattr(paged._OnDevice, "_on", lambda self, stream: 0)
    monkeypatch.setattr(paged._OnDevice, "_scratch", lambda self, n, sp: torch.empty(n, dtype=torch.uint8))
    for code, error in ((L.MOE_EINVAL, ValueError), (L.MOE_EUNSUP, ValueError), (L.MOE_EHIP, L.MoeError)):
        class Refuses:
            def __getattr__(self, name):
                return getattr(lib, name) if "last_error" in name or name.endswith("_size") else lambda *a: code

        with monkeypatch.context() as p:
            p.setattr(paged.L, "lib", Refuses)
            c, a = cpu_cache(), ok_args()
            for call in calls(c, a).values():
                with pytest.raises(error):
                    call()
            table = PageTable.new(3, 4, 9, 32, "cpu")
            with pytest.raises(error):
                table.advance(torch.zeros(3, dtype=torch.int32), Rows.new(3, 5, "cpu"))


def test_what_addresses_are_taken_of_is_not_replaced(lib):
    """The kernels work on the tensors an object was made with: another one
    in their place would not be seen, so it is refused."""
    c, t, r = cpu_cache(), PageTable.new(3, 4, 9, 32, "cpu"), Rows.new(3, 5, "cpu")
    for x, names in ((c, ("pool", "table", "means", "n_kv", "qd", "vd", "page", "n_pages", "c", "device")),
                     (t, ("table", "length", "ring", "state", "page", "device")),
                     (r, ("row_start", "seq", "pos", "slot", "status", "n_seq", "device"))):
        for name in names:
            now = getattr(x, name)
            with pytest.raises(AttributeError):
                setattr(x, name, now)
            assert getattr(x, name) is now
    t.length.fill_(3)  # their contents are the caller's
    assert t.length.tolist() == [3, 3, 3]
