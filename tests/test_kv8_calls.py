"""The 8-bit cache's, the 8-bit product's and the head rotation's entry points
on the CPU: what they refuse, before anything is queued, and their sizes."""
import ctypes as C

import pytest
import torch

from moe_amd import _lib as L
from moe_amd.heads import HeadRope
from moe_amd.int8 import Int8Linear
from moe_amd.paged import KvCache8, Rows

P = 0x10000  # an address that no refused call reads


@pytest.fixture(scope="module")
def lib():
    if not L.LIB_PATH.exists():
        from moe_amd.build import build

        build()
    return L.lib()


def kv8(**kw):
    c = dict(codes=P, scales=P, open=P, table=P, codes_bytes=1 << 40, scales_bytes=1 << 40, open_bytes=1 << 40, n_seq=4,
             max_pages=10, n_pages=100, page=64, n_kv=2, qd=64, vd=64)
    c.update(kw)
    return L.Kv8C(**c)


BAD_CACHES = [dict(codes=None), dict(scales=None), dict(open=None), dict(table=None), dict(codes=P + 8), dict(scales=P + 4),
              dict(open=P + 8), dict(codes_bytes=100 * 2 * 64 * 128 - 1), dict(scales_bytes=100 * 2 * 32 - 1),
              dict(open_bytes=4 * 2 * (128 * 128 + 32) - 1), dict(n_seq=0), dict(max_pages=0), dict(n_pages=0), dict(n_kv=0),
              dict(n_kv=65536), dict(page=32), dict(page=96), dict(page=8192), dict(page=0), dict(page=4096, max_pages=1 << 20),
              dict(qd=0), dict(qd=48), dict(vd=288), dict(vd=-32), dict(n_pages=2 ** 31 - 1, page=4096, n_kv=65535)]


def attention(lib, c, q=P, stride=512, rows=3, heads=8, seq=P, pos=P, max_pos=100, window=0, out=P, ws=P, ws_bytes=1 << 40):
    return lib.moe_kv8_attention(C.byref(c), q, stride, rows, heads, 0.125, seq, pos, max_pos, window, out, stride, ws, ws_bytes,
                                 None)


def store(lib, c, k=P, v=P, rows=3, row_start=P, seq=P, pos=P, slots=P):
    return lib.moe_kv8_store(C.byref(c), k, 128, v, 128, rows, row_start, seq, pos, slots, None)


def load(lib, c, slots=P, rows=3):
    return lib.moe_kv8_load(C.byref(c), slots, rows, P, 128, P, 128, None)


@pytest.mark.parametrize("call", [attention, store, load])
@pytest.mark.parametrize("bad", BAD_CACHES, ids=str)
def test_refuses_bad_caches(lib, call, bad):
    assert call(lib, kv8(**bad)) in (L.MOE_EINVAL, L.MOE_EUNSUP)
    assert lib.moe_last_error()


@pytest.mark.parametrize("call", [attention, store, load])
def test_no_rows_are_no_work(lib, call):
    """Null pointers and all: torch's empty tensors have no address."""
    kw = {attention: dict(q=None, seq=None, pos=None, out=None), load: dict(slots=None),
          store: dict(k=None, v=None, row_start=None, seq=None, pos=None, slots=None)}[call]
    assert call(lib, kv8(), rows=0, **kw) == L.MOE_OK
    assert call(lib, kv8(), rows=-1) == L.MOE_EINVAL
    for k in kw:
        assert call(lib, kv8(), **{k: None}) == L.MOE_EINVAL


@pytest.mark.parametrize("bad", [dict(heads=7), dict(heads=0), dict(heads=-2), dict(max_pos=-1), dict(max_pos=640)], ids=str)
def test_attention_refuses(lib, bad):
    assert attention(lib, kv8(), **bad) == L.MOE_EINVAL
    size = {k: bad.get(k, v) for k, v in dict(rows=3, heads=8, max_pos=100, window=0).items()}
    assert lib.moe_kv8_attention_workspace_size(C.byref(kv8()), *size.values(), C.byref(C.c_uint64())) == L.MOE_EINVAL


@pytest.mark.parametrize("rows", [2 ** 24 - 255, 2 ** 31 - 1])
def test_refuses_more_rows_than_a_launch(lib, rows):
    for call in (store, load):
        assert call(lib, kv8(), rows=rows) == L.MOE_EUNSUP


def test_sizes():
    assert KvCache8.sizes(3, 5, n_kv=2, qd=64, vd=96, page=128) == (3 * 2 * 128 * 160, 3 * 2 * 2 * 32, 5 * 2 * (128 * 160 + 32))
    for bad in (dict(n_kv=0), dict(qd=40), dict(page=16), dict(vd=512)):
        with pytest.raises(ValueError):
            KvCache8.sizes(3, 5, **{**dict(n_kv=2, qd=64, vd=96, page=128), **bad})
    with pytest.raises(ValueError):
        KvCache8.sizes(2 ** 31, 5, n_kv=2, qd=64, vd=96, page=128)
    with pytest.raises(ValueError):
        KvCache8.sizes(3, 2 ** 32 + 5, n_kv=2, qd=64, vd=96, page=128)


def rows_of(n, n_seq=2):
    z = lambda k, t=torch.int32: torch.zeros(k, dtype=t)  # noqa: E731
    return Rows(z(n_seq + 1), z(n), z(n), z(n, torch.int64), z(n_seq))


def test_cache_object_refuses():
    kw = dict(n_kv=2, qd=64, vd=64, page=64)
    table = torch.zeros((2, 3), dtype=torch.int32)
    c = KvCache8.new(4, table, **kw)
    a = (c.codes, c.scales, c.open_blocks, table)
    for i, bad in ((0, c.codes[:100]), (0, c.codes.float()), (1, c.scales[:-1]), (1, c.scales.view(-1, 2)), (2, c.open_blocks[:-1]),
                   (2, c.open_blocks.view(torch.int8)), (3, table.long()), (3, table[0])):
        with pytest.raises(ValueError):
            KvCache8(*a[:i], bad, *a[i + 1:], **kw)
    with pytest.raises(AttributeError):
        c.codes = c.codes.clone()
    f = torch.zeros
    for k, v, rows in ((f(3, 64), f(3, 128), rows_of(3)), (f(3, 128), f(4, 128), rows_of(3)), (f(3, 128), f(3, 128), rows_of(4)),
                       (f(3, 128).half(), f(3, 128), rows_of(3)), (f(3, 128), f(3, 128), rows_of(3, n_seq=3)),
                       (f(3, 128), f(3, 128), rows_of(3))):  # (the last: tensors on the CPU)
        with pytest.raises(ValueError):
            c.store(k, v, rows)
    i = torch.zeros(3, dtype=torch.int32)
    for q, seq, pos, out, max_pos, window in (
            (f(3, 100), i, i, f(3, 128), 5, 0), (f(3, 192), i, i, f(3, 192), 5, 0), (f(3, 128), i.long(), i, f(3, 128), 5, 0),
            (f(3, 128), i, i[:2], f(3, 128), 5, 0), (f(3, 128), i, i, f(3, 64), 5, 0), (f(3, 128), i, i, f(3, 128), 192, 0),
            (f(3, 128), i, i, f(3, 128), -1, 0), (f(3, 128), i, i, f(3, 128), 5, 2 ** 32 + 16), (f(3, 128), i, i, f(3, 128), 5, 0)):
        with pytest.raises(ValueError):
            c.attend(q, seq, pos, out, max_pos=max_pos, scale=1.0, window=window)
    for slots, k, v in ((i, f(3, 128), None), (i.long(), f(3, 64), None), (i.long(), None, f(2, 128)), (i.long(), f(3, 128), None)):
        with pytest.raises(ValueError):
            c.load(slots, k, v)


# ----------------------------------------------------------------- products


def product(lib, packed=P, n=64, k=128, x=P, xs=128, t=3, y=P, ys=64, res=None, rs=0, ws=P, ws_bytes=1 << 40):
    return lib.moe_int8_linear(packed, n, k, x, xs, t, y, ys, res, rs, ws, ws_bytes, None)


def pack(lib, w=P, dt=L.DT_F32, row_bytes=512, rows=64, row0=0, n=64, k=128, packed=P, size=1 << 40):
    return lib.moe_int8_pack(w, dt, row_bytes, rows, row0, n, k, packed, size, None)


@pytest.mark.parametrize("bad", [dict(packed=None), dict(packed=P + 16), dict(x=None), dict(y=None), dict(n=0), dict(k=0),
                                 dict(t=-1), dict(t=2 ** 20 + 1), dict(ws=None), dict(ws=P + 128), dict(ws_bytes=2000),
                                 dict(k=131073), dict(n=2 ** 24), dict(n=2 ** 24 + 1)], ids=str)
def test_product_refuses(lib, bad):
    assert product(lib, **bad) in (L.MOE_EINVAL, L.MOE_EUNSUP)
    assert lib.moe_last_error()


def test_product_of_no_rows(lib):
    assert product(lib, t=0, packed=None, x=None, y=None, ws=None, ws_bytes=0) == L.MOE_OK


@pytest.mark.parametrize("bad", [dict(w=None), dict(packed=None), dict(packed=P + 64), dict(rows=-1), dict(row0=-1), dict(row0=1),
                                 dict(dt=7), dict(dt=L.DT_Q6_REF), dict(dt=L.DT_Q4_0, k=100, row_bytes=1000), dict(row_bytes=511),
                                 dict(size=64 * 128 + 255), dict(k=131073, row_bytes=1 << 20)], ids=str)
def test_pack_refuses(lib, bad):
    assert pack(lib, **bad) in (L.MOE_EINVAL, L.MOE_EUNSUP)


def test_pack_size(lib):
    b = C.c_uint64()
    for n, k, want in ((64, 128, 64 * 128 + 256), (1, 1, 16 * 64 + 64), (17, 65, 32 * 128 + 128)):
        assert lib.moe_int8_pack_size(n, k, C.byref(b)) == L.MOE_OK and b.value == want
    assert lib.moe_int8_pack_size(0, 4, C.byref(b)) == L.MOE_EINVAL
    assert lib.moe_int8_linear_workspace_size(64, 128, -1, C.byref(b)) == L.MOE_EINVAL


def test_product_object_refuses():
    w = torch.zeros(8, 16)
    for bad in ([], [w, torch.zeros(8, 15)], w.int(), w.t(), torch.zeros(8), torch.zeros(0, 16), torch.zeros(8, 0), w.expand(2, 8, 16),
                torch.zeros(1, 16).expand(8, 16), torch.zeros(1, 131073), w):  # (the last: on the CPU)
        with pytest.raises(ValueError):
            Int8Linear(bad)


# ------------------------------------------------------------------- heads


def rope(lib, q=P, k=P, v=None, rows=3, pos=P, qo=P, ko=P, vo=None, **kw):
    h = dict(inv_freq=P, heads=8, n_kv=2, width=64, q_span=1, k_span=1, offset=0, dim=64, n_inv=32, eps=1e-6)
    h.update(kw)
    return lib.moe_head_rope_rows(C.byref(L.HeadRopeC(**h)), q, 512, k, 128, v, 128, rows, pos, qo, 512, ko, 128, vo, 128, None)


@pytest.mark.parametrize("bad", [dict(q=None), dict(k=None), dict(pos=None), dict(qo=None), dict(ko=None), dict(rows=-1),
                                 dict(rows=2 ** 24), dict(heads=0), dict(n_kv=0), dict(heads=30001), dict(width=0), dict(dim=-2),
                                 dict(dim=63), dict(offset=2), dict(offset=-2, dim=2), dict(n_inv=-1), dict(inv_freq=None),
                                 dict(q_span=2), dict(k_span=0), dict(v=P, v_width=64), dict(v=P, vo=P, v_width=0),
                                 dict(offset=2 ** 31 - 1, dim=64)], ids=str)
def test_heads_refuse(lib, bad):
    assert rope(lib, **bad) in (L.MOE_EINVAL, L.MOE_EUNSUP)
    assert lib.moe_last_error()


def test_heads_of_no_rows(lib):
    assert rope(lib, rows=0, q=None, k=None, pos=None, qo=None, ko=None) == L.MOE_OK


def test_heads_object_refuses():
    inv, one = torch.ones(32), torch.ones(64)
    for bad in (dict(dim=66), dict(dim=63), dict(offset=2, dim=64), dict(offset=-1), dict(q_norm=one[:60]), dict(k_norm=torch.ones(2, 64)),
                dict(q_norm=one.double()), dict(k_norm=torch.ones(512)), dict(q_bias=one), dict(k_bias=torch.ones(512)),
                dict(v_bias=torch.ones(0)), dict(q_norm=torch.ones(128)[::2])):
        with pytest.raises(ValueError):
            HeadRope(8, 2, 64, inv, **bad)
    for shape in ((0, 2, 64), (8, 0, 64), (8, 2, 0), (2 ** 32 + 8, 2, 64)):
        with pytest.raises(ValueError):
            HeadRope(*shape, inv)
    h = HeadRope(8, 2, 64, inv)
    f, i = torch.zeros, torch.zeros(3, dtype=torch.int32)
    for args, kw in (((f(3, 511), f(3, 128), i), {}), ((f(3, 512), f(3, 64), i), {}), ((f(3, 512), f(4, 128), i), {}),
                     ((f(3, 512), f(3, 128), i.long()), {}), ((f(3, 512), f(3, 128), i[:2]), {}),
                     ((f(3, 512), f(3, 128), i), dict(q_out=f(3, 500))), ((f(3, 512), f(3, 128), i, f(3, 128)), dict(v_out=f(3, 128))),
                     ((f(3, 512), f(3, 128), i), {})):  # (the last: tensors on the CPU)
        with pytest.raises(ValueError):
            h(*args, **kw)
    with pytest.raises(AttributeError):
        h.inv_freq = inv.clone()
