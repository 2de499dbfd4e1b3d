"""The paged 4-bit cache on the GPU (moe_pages_advance, moe_kv4_*) against the
plain 64-bit forms of kv4_reference.py.

Tolerance of attention.  A block's product is a sum of 32 products of exact
codes with a query in two f16 pieces or f32 (relative error up to 2^-22 of the
row's largest query), scaled and added up in f32: a score of qd values has an
error of about sqrt(qd) 2^-22 times its terms' size, a relative error of its
weight of below 2e-6 for the scores of order 1 here; outputs average values of
order 1 under such weights.  gpu_util.TOL = 5e-6 of the largest output is the
bar of moe_attention on the same quantities.  Larger scores carry larger
errors in proportion; the tests that make them say so."""
import math

import numpy as np
import pytest

import kv4_reference as ref
from gpu_util import TOL

pytestmark = pytest.mark.gpu

HEADS = [(8, 2, 64, 64), (16, 16, 192, 128), (32, 8, 128, 128), (6, 2, 96, 96), (40, 1, 64, 32), (4, 2, 256, 256),
         (3, 3, 32, 160), (48, 2, 128, 128), (1, 1, 224, 64)]
# name: (sequence, position) of each row
ROWS = {
    "decode": [(s, p) for s, p in enumerate([0, 15, 16, 31, 32, 33, 130, 63, 64, 1, 299])],
    "one_row": [(0, 200)],
    "first": [(0, 0)],
    "prompt": [(0, p) for p in range(37)],
    "chunk": [(0, 100 + p) for p in range(70)],
    "mixed": [(0, p) for p in range(9)] + [(1, 40 + p) for p in range(21)] + [(2, 5), (3, 77)] +
             [(0, 9 + p) for p in range(13)] + [(1, -1), (-1, 3), (9, 3)],
    "shuffled": [(0, p) for p in (90, 3, 50, 51, 7, 0, 128)],
}


def filled(shape, n_seq, ctx, page, seed=0, spread=0.0, spare=2):
    """A pool whose sequences hold ctx positions of N(0, 1) keys and values
    on scattered pages, written by the reference; (Pool, table)."""
    heads, n_kv, qd, vd = shape
    g = np.random.default_rng(seed)
    mp = -(-ctx // page)
    pool = ref.Pool(n_seq * mp + spare, n_kv, qd, vd, page)
    table = g.permutation(pool.n_pages)[:n_seq * mp].reshape(n_seq, mp).astype(np.int32)
    size = (n_seq, mp * page)
    k = g.standard_normal((*size, n_kv, qd)).astype(np.float32) * np.exp(spread * g.standard_normal((*size, 1, 1))).astype(np.float32)
    v = g.standard_normal((*size, n_kv, vd)).astype(np.float32) * np.exp(spread * g.standard_normal((*size, 1, 1))).astype(np.float32)
    for x, keys in ((k, True), (v, False)):
        code, h = ref.quantise(x)
        for s in range(n_seq):
            for p in range(mp * page):
                for kv in range(n_kv):
                    pool.put(table[s, p // page] * page + p % page, kv, code[s, p, kv], h[s, p, kv], keys)
    return pool, table


_filled = {}


def shared(shape, n_seq, ctx, page):
    """filled(), kept for the tests that leave it alone."""
    key = (shape, n_seq, ctx, page)
    if key not in _filled:
        _filled.clear()
        _filled[key] = filled(*key)
    return _filled[key]


def on_gpu(pool, table, means=None):
    import torch

    from moe_amd.paged import KvCache

    d = lambda x: torch.from_numpy(np.ascontiguousarray(x)).cuda()  # noqa: E731
    return KvCache(d(pool.raw), d(table), n_kv=pool.n_kv, qd=pool.qd, vd=pool.vd, page=pool.page,
                   means=None if means is None else d(means))


def ints(v, t="int32"):
    import torch

    return torch.tensor([int(x) for x in v], dtype=getattr(torch, t), device="cuda")


def run_attend(cache, q, seq, pos, heads, scale, window=0, lists=None, fill=7.0, max_pos=None, **kw):
    import torch

    out = torch.full((len(seq), heads * cache.vd), fill, device="cuda")
    cache.attend(torch.from_numpy(q).cuda(), ints(seq), ints(pos), out, max_pos=max(max(pos), 0) if max_pos is None else max_pos,
                 scale=scale, window=window, pages=None if lists is None else torch.from_numpy(lists).cuda(), **kw)
    torch.cuda.synchronize()
    return out.cpu().numpy()


def close(got, want, tol=TOL):
    big = np.abs(want).max()
    err = np.abs(got - want).max() / (big if big > 0 else 1.0)
    assert err < tol, err


# ----------------------------------------------------------------- the tables


def run_advance(length, add, table, ring, state, page, max_rows, separate):
    import torch

    from moe_amd.paged import PageTable, Rows

    t, r = torch.from_numpy(table).cuda(), torch.from_numpy(ring).cuda()
    pt = PageTable(t, ints(length), r, ints(state), page)
    rows = Rows.new(len(length), max_rows, "cuda")
    out = PageTable(t, ints([-7] * len(length)), r, ints([-7, -7]), page) if separate else pt
    pt.advance(ints(add), rows, out=out if separate else None)
    torch.cuda.synchronize()
    c = lambda x: x.cpu().numpy()  # noqa: E731
    if separate:
        assert c(pt.length).tolist() == list(length) and c(pt.state).tolist() == list(state)
    return dict(length=c(out.length), state=c(out.state), row_start=c(rows.row_start), seq=c(rows.seq), pos=c(rows.pos),
                slot=c(rows.slot), status=c(rows.status)), c(t), c(r)


@pytest.mark.parametrize("separate", [False, True])
@pytest.mark.parametrize("n,page,max_pages,max_rows,free", [
    (1, 32, 1, 1, 1), (1, 64, 40, 2500, 100), (5, 32, 7, 40, 3), (32, 64, 64, 32, 50), (1000, 64, 20, 3000, 90),
    (1024, 32, 9, 1500, 2000), (1025, 128, 6, 1400, 60), (5000, 64, 10, 7000, 700), (300, 4096, 3, 9000, 20),
    (7, 32, 30, 0, 9)])
def test_advance(n, page, max_pages, max_rows, free, separate):
    """Sequences of every kind: growing by one, by a prompt, idle, ended, too
    long, more than the rows or pages there are; negative and too large lengths."""
    g = np.random.default_rng(n + page)
    cap = max_pages * page
    length = g.integers(0, cap + 1, n)
    add = np.where(g.random(n) < 0.1, g.integers(0, max(2, max_rows // 4), n), 1)
    add[g.random(n) < 0.1] = -1
    add[g.random(n) < 0.1] = 0
    length[g.random(n) < 0.02] = -5
    length[g.random(n) < 0.02] = cap + 9
    add[g.random(n) < 0.01] = 2 ** 31 - 1
    length, add = length.astype(np.int32), add.astype(np.int32)
    n_pages = n * max_pages + free
    ids = g.permutation(n_pages).astype(np.int32)
    table = ids[:n * max_pages].reshape(n, max_pages).copy()
    head = int(g.integers(0, n_pages))
    ring = np.full(n_pages, -9, np.int32)
    ring[(head + np.arange(free)) % n_pages] = ids[n * max_pages:]
    state = np.array([head, free], np.int32)
    t, r = table.copy(), ring.copy()
    want = ref.advance(length, add, t, r, state, page, max_rows)
    got, gt, gr = run_advance(length, add, table, ring, state, page, max_rows, separate)
    for k, v in want.items():
        assert np.array_equal(got[k], np.asarray(v)), k
    assert np.array_equal(gt, t) and np.array_equal(gr, r)


def test_advance_over_many_steps():
    """A server's life: sequences grow, end and are given others' pages; no
    page is held twice and none is lost."""
    import torch

    from moe_amd.paged import PageTable, Rows

    g = np.random.default_rng(1)
    n, page, mp, pages = 40, 32, 12, 150
    pt, rows = PageTable.new(n, mp, pages, page, "cuda"), Rows.new(n, 300, "cuda")
    length, state = np.zeros(n, np.int32), np.array([0, pages], np.int32)
    table, ring = np.full((n, mp), -1, np.int32), np.arange(pages, dtype=np.int32)
    for step in range(60):
        add = np.where(g.random(n) < 0.1, g.integers(1, 120, n), 1)
        add[g.random(n) < 0.08] = -1
        add = add.astype(np.int32)
        want = ref.advance(length, add, table, ring, state, page, 300)
        length, state = want["length"], want["state"]
        pt.advance(torch.from_numpy(add).cuda(), rows)
        assert pt.length.cpu().numpy().tolist() == length.tolist()
        assert pt.state.cpu().numpy().tolist() == state.tolist()
        assert rows.slot.cpu().numpy().tolist() == want["slot"]
        t, r = pt.table.cpu().numpy(), pt.ring.cpu().numpy()
        held = [x for i in range(n) for x in t[i, :-(-length[i] // page)]]
        free = [r[(state[0] + j) % pages] for j in range(state[1])]
        assert sorted(held + free) == list(range(pages))


# ------------------------------------------------------------ rows in and out


@pytest.mark.parametrize("shape", HEADS, ids=str)
@pytest.mark.parametrize("page", [32, 64, 256])
def test_store_and_load(shape, page):
    """Bytes of the pool, means and rows read back, of scattered and of
    consecutive slots, some rows skipped, rows apart in memory."""
    import torch

    heads, n_kv, qd, vd = shape
    g = np.random.default_rng(page)
    n_pages = 5
    pool = ref.Pool(n_pages, n_kv, qd, vd, page, g.integers(0, 255, n_pages * n_kv * page // 32 * 18 * (qd + vd)).astype(np.uint8))
    start = int(g.integers(0, page))
    slots = np.r_[start + np.arange(page), g.permutation(page)[:9] + 3 * page, [4 * page + page - 1, -1, n_pages * page, 2 ** 40]]
    k = (g.standard_normal((len(slots), n_kv * qd)) * np.exp(3 * g.standard_normal((len(slots), 1)))).astype(np.float32)
    v = (g.standard_normal((len(slots), n_kv * vd)) * np.exp(3 * g.standard_normal((len(slots), 1)))).astype(np.float32)
    k[0, :32], v[1, :32] = 0, -0.0
    k[2, :32] = np.linspace(-3.5, 3.5, 32)  # halves: rounded away from zero
    before = pool.raw.copy()
    means = g.standard_normal((n_pages, n_kv, qd)).astype(np.float16)
    cache = on_gpu(pool, np.zeros((1, 1), np.int32), means)
    wide = lambda x: torch.from_numpy(np.concatenate([x, np.full((len(x), 5), np.nan, np.float32)], 1)).cuda()[:, :x.shape[1]]  # noqa: E731
    cache.store(wide(k), wide(v), ints(slots, "int64"))
    pool.store(slots, k, v)
    assert np.array_equal(cache.pool.cpu().numpy(), pool.raw) and not np.array_equal(before, pool.raw)
    for p in range(n_pages):
        if p * page + page - 1 in slots:
            means[p] = pool.mean(p)
    got = cache.means.cpu().numpy()
    same = (got.view(np.uint16) == means.view(np.uint16)) | (np.isnan(got) & np.isnan(means))
    assert same.all()
    kb, vb = torch.full((len(slots), n_kv * qd + 3), 5.0, device="cuda"), torch.full((len(slots), n_kv * vd), 5.0, device="cuda")
    cache.load(ints(slots, "int64"), kb[:, :n_kv * qd], vb)
    kb, vb = kb.cpu().numpy(), vb.cpu().numpy()
    assert (kb[:, n_kv * qd:] == 5).all()
    for r, s in enumerate(slots):
        if not 0 <= s < n_pages * page:
            assert (kb[r] == 5).all() and (vb[r] == 5).all()
            continue
        for kv in range(n_kv):
            assert np.array_equal(kb[r, kv * qd:(kv + 1) * qd], pool.get(s, kv, True).astype(np.float32))
            assert np.array_equal(vb[r, kv * vd:(kv + 1) * vd], pool.get(s, kv, False).astype(np.float32))


@pytest.mark.parametrize("page", [32, 64])
def test_store_runs_of_rows(page):
    """Runs that begin at any offset, follow one another, break off, go
    backwards: rows that are written four at a time beside single ones."""
    n_kv, qd, vd = 1, 64, 96
    g = np.random.default_rng(page)
    for trial in range(6):
        n_pages = [6, 300, 400, 5, 350, 320][trial] * 32 // page  # few rows, and enough for the kernel of four
        free = g.permutation(n_pages * page // 8)
        slots = []
        for b in free[:len(free) - 2]:
            run = list(range(b * 8, b * 8 + 8))
            how = int(g.integers(0, 5))
            slots += [run, run[int(g.integers(0, 8)):], run[::-1], run[:int(g.integers(1, 8))],
                      [run[i] for i in g.permutation(8)]][how]
            if g.random() < 0.2:
                slots.append(-1)
        k = g.standard_normal((len(slots), n_kv * qd)).astype(np.float32)
        v = g.standard_normal((len(slots), n_kv * vd)).astype(np.float32)
        pool = ref.Pool(n_pages, n_kv, qd, vd, page, g.integers(0, 255, n_pages * n_kv * page // 32 * 18 * (qd + vd)).astype(np.uint8))
        cache = on_gpu(pool, np.zeros((1, 1), np.int32))
        import torch

        cache.store(torch.from_numpy(k).cuda(), torch.from_numpy(v).cuda(), ints(slots, "int64"))
        pool.store(slots, k, v)
        assert np.array_equal(cache.pool.cpu().numpy(), pool.raw)


def test_store_as_the_host_quantiser():
    """Codes and scales equal moe_quantize_rows(Q4_0)'s, over the range of
    f32: subnormal and overflowing scales, zeros, infinities, NaNs."""
    import ctypes as C

    import torch

    from moe_amd import _lib as L
    from moe_amd.paged import KvCache

    g = np.random.default_rng(3)
    n, d = 512, 64
    x = (g.standard_normal((n, d)) * np.exp2(g.uniform(-40, 22, (n, 1)))).astype(np.float32)
    x[0], x[1] = 0, -0.0
    x[2, 3], x[3, 40], x[4, 1], x[5, :] = np.inf, -np.inf, np.nan, np.nan
    x[6, :32] = 3.4e38
    raw = np.empty((n, d // 32, 18), np.uint8)
    L.check(L.lib().moe_quantize_rows(L.DT_Q4_0, x.ctypes.data_as(C.c_void_p), n, d, raw.ctypes.data_as(C.c_void_p)))
    scale = raw[..., :2].copy().view(np.float16)[..., 0]
    codes = np.concatenate([raw[..., 2:] & 15, raw[..., 2:] >> 4], -1).reshape(n, d)
    want = ref.value(codes, scale).astype(np.float32)
    cache = KvCache.new(n // 32, ints([0]).view(1, 1), n_kv=1, qd=d, vd=d, page=32)
    xs, slots = torch.from_numpy(x).cuda(), torch.arange(n, device="cuda")
    cache.store(xs, xs, slots)
    k, v = torch.empty_like(xs), torch.empty_like(xs)
    cache.load(slots, k, v)
    for got in (k.cpu().numpy(), v.cpu().numpy()):
        assert np.array_equal(got, want, equal_nan=True)
    p = ref.Pool(n // 32, 1, d, d, 32, cache.pool.cpu().numpy())
    for r in range(n):
        at, i = p._at(r, 0)
        sb = p._bytes(i, True)[1]
        got = np.stack([p.raw[at + sb], p.raw[at + sb + 1]], -1).copy().view(np.float16)[..., 0]
        assert np.array_equal(got.view(np.uint16), scale[r].view(np.uint16))


# ------------------------------------------------------------------ attention


@pytest.mark.parametrize("shape", HEADS, ids=str)
@pytest.mark.parametrize("page", [32, 128])
def test_attention(shape, page):
    heads, n_kv, qd, vd = shape
    pool, table = shared(shape, 11, 300, page)
    cache = on_gpu(pool, table)
    for name, rows in ROWS.items():
        seq, pos = zip(*rows)
        q = np.random.default_rng(len(rows)).standard_normal((len(rows), heads * qd)).astype(np.float32)
        for window in (0, 21):
            scale = 1.0 / math.sqrt(qd)
            got = run_attend(cache, q, seq, pos, heads, scale, window)
            want = ref.attend(pool, table, q, seq, pos, heads, scale, window, out=np.full(got.shape, 7.0))
            close(got, want)
            for r, (s, p) in enumerate(rows):
                if p < 0 or not 0 <= s < len(table):
                    assert (got[r] == 7).all(), "a row that is none was written"


def lists_of(g, rows, n_kv, n_sel, mp):
    """Ascending lists with holes: short ones, an empty one, unsorted and
    repeated entries, pages behind the table's end."""
    out = np.full((rows, n_kv, n_sel), -1, np.int32)
    for r in range(rows):
        for kv in range(n_kv):
            k = int(g.integers(0, min(n_sel, mp) + 1))
            out[r, kv, :k] = np.sort(g.permutation(mp)[:k])
    out[0, 0, :] = -1
    if n_sel > 2:
        out[-1, -1, :3] = [1, 1, 0]
        out[-1, 0, -1] = mp + 5
    return out


@pytest.mark.parametrize("shape", HEADS, ids=str)
@pytest.mark.parametrize("n_sel", [1, 3, 9])
def test_attention_over_lists(shape, n_sel):
    heads, n_kv, qd, vd = shape
    pool, table = shared(shape, 11, 300, 32)
    cache = on_gpu(pool, table)
    g = np.random.default_rng(n_sel)
    for name in ("decode", "one_row", "chunk", "mixed"):
        seq, pos = zip(*ROWS[name])
        q = g.standard_normal((len(seq), heads * qd)).astype(np.float32)
        lists = lists_of(g, len(seq), n_kv, n_sel, table.shape[1])
        for window in (0, 70):
            got = run_attend(cache, q, seq, pos, heads, qd ** -0.5, window, lists)
            want = ref.attend(pool, table, q, seq, pos, heads, qd ** -0.5, window, lists, np.full(got.shape, 7.0))
            close(got, want)


def test_rows_that_see_nothing():
    """Pages that hold nothing (outside the pool), in part and altogether."""
    shape = (8, 2, 64, 64)
    pool, table = shared(shape, 11, 300, 32)
    bad = table.copy()
    bad[0], bad[1, 0], bad[2, 3], bad[3, -1] = -1, pool.n_pages, 2 ** 31 - 1, -(2 ** 31)
    rows = [(0, 200), (1, 10), (1, 40), (2, 250), (3, 299), (4, 60)]
    seq, pos = zip(*rows)
    q = np.random.default_rng(0).standard_normal((6, 8 * 64)).astype(np.float32)
    got = run_attend(on_gpu(pool, bad), q, seq, pos, 8, 0.125)
    close(got, ref.attend(pool, bad, q, seq, pos, 8, 0.125, out=np.full(got.shape, 7.0)))
    assert (got[0] == 0).all() and (got[1] == 0).all()


@pytest.mark.parametrize("shape", [(8, 2, 64, 64), (16, 16, 192, 128), (6, 2, 96, 96), (4, 2, 256, 256)], ids=str)
@pytest.mark.parametrize("bad", [0x7c00, 0x7e00, 0xfc00])
def test_unseen_positions_do_not_matter(shape, bad):
    """Scales that are infinite or NaN, at positions before the window, after
    the row and in a page's rest, leave a row as it was; a row that sees one is
    not finite."""
    heads, n_kv, qd, vd = shape
    pool, table = filled(shape, 1, 100, 32)
    seq, pos = [0] * 30, list(range(50, 80))
    # what lies beside the positions in question is larger than all else
    for p in (27, 64, 67):
        for kv in range(n_kv):
            code = np.random.default_rng(p).integers(1, 16, vd).astype(np.uint8)
            pool.put(int(table[0, p // 32]) * 32 + p % 32, kv, code, np.full(vd // 32, 3e4, np.float16), False)
    q = np.random.default_rng(1).standard_normal((30, heads * qd)).astype(np.float32)
    want = ref.attend(pool, table, q, seq, pos, heads, qd ** -0.5, 25)
    at = (0, 10, 25, 26, 65, 66, 79, 80, 99)
    for p in at:
        slot = int(table[0, p // 32]) * 32 + p % 32
        for kv in range(n_kv):
            for keys, d in ((True, qd), (False, vd)):
                code = np.random.default_rng(p).integers(1, 16, d).astype(np.uint8)
                pool.put(slot, kv, code, np.full(d // 32, bad, np.uint16).view(np.float16), keys)
    got = run_attend(on_gpu(pool, table), q, seq, pos, heads, qd ** -0.5, 25)
    sees = np.array([any(max(0, p - 24) <= b <= p for b in at) for p in pos])
    assert (~sees).sum() >= 3 and sees.any()
    close(got[~sees], want[~sees])
    assert not np.isfinite(got[sees]).all(axis=1).any()


@pytest.mark.parametrize("heads", [32, 64])
def test_unseen_positions_do_not_matter_to_many_rows(heads):
    """The same where the rows fill the wide groups: 600 rows, an infinity and
    a NaN at positions that the earlier rows do not see, in tiles the others'
    scales follow at once."""
    shape = (heads, 8, 128, 128)
    cache, k, v = device_pool(shape, 1, 640, 64)
    import torch

    q = torch.randn((600, heads * 128), generator=torch.Generator(device="cuda").manual_seed(3), device="cuda")
    seq, pos = [0] * 600, list(range(600))
    clean = run_attend(cache, q.cpu().numpy(), seq, pos, heads, 128 ** -0.5)
    pick = list(range(0, 600, 17)) + [399, 400, 401, 431, 432]
    close(clean[pick], attend64(k, v, q[pick], [0] * len(pick), pick, heads, 128 ** -0.5))
    pool = ref.Pool(10, 8, 128, 128, 64, cache.pool.cpu().numpy().copy())
    table = cache.table.cpu().numpy()
    bad = np.array([np.inf, 1, np.nan, -np.inf], np.float16)
    for p in (400, 431):
        slot = int(table[0, p // 64]) * 64 + p % 64
        for kv in range(8):
            for keys in (True, False):
                pool.put(slot, kv, np.full(128, 11, np.uint8), bad, keys)
    cache.pool.copy_(torch.from_numpy(pool.raw))
    got = run_attend(cache, q.cpu().numpy(), seq, pos, heads, 128 ** -0.5)
    # The finite scale beside them (1, above every other) moves the power of two
    # that the weights are held under, so their two pieces round elsewhere: by
    # up to 2^-22 of a weight, within TOL.
    close(got[:400], clean[:400])
    assert not np.isfinite(got[400:]).all(axis=1).any()


def test_large_and_small_values():
    """Values from 1e-6 to 1e5 in one cache, scores hundreds apart."""
    shape = (8, 2, 64, 64)
    pool, table = filled(shape, 2, 200, 64, seed=5, spread=3.0)
    seq, pos = [0] * 39 + [1], list(range(150, 189)) + [191]
    q = np.random.default_rng(2).standard_normal((40, 8 * 64)).astype(np.float32)
    got = run_attend(on_gpu(pool, table), q, seq, pos, 8, 0.125)
    want = ref.attend(pool, table, q, seq, pos, 8, 0.125)
    # Scores reach several thousand: a relative error of 2^-22 of one is 1e-3
    # of its weight where two of them compete.
    assert np.isfinite(got).all()
    scores = 64 ** 0.5 * 0.125 * np.exp(3.0 * 3) * 8
    close(got, want, max(TOL, scores * 2.0 ** -22 * 4))


@pytest.mark.parametrize("tiny", [1e-7, 6e-5, 1.0, 6e4])
def test_scales_over_their_range(tiny):
    """All of a head's values of one size, from subnormal f16 scales up to the
    largest: outputs keep their relative precision."""
    shape = (8, 2, 64, 64)
    heads, n_kv, qd, vd = shape
    pool, table = filled(shape, 1, 150, 32, seed=9)
    p = pool.raw.reshape(-1, pool.tile)
    h = np.random.default_rng(0).uniform(0.5, 1.0, (len(p), vd)).astype(np.float64) * tiny
    p[:, 18 * qd + 16 * vd:] = h.astype(np.float16).view(np.uint8).reshape(len(p), -1)
    seq, pos = [0] * 20, list(range(120, 140))
    q = np.random.default_rng(3).standard_normal((20, heads * qd)).astype(np.float32)
    got = run_attend(on_gpu(pool, table), q, seq, pos, heads, 0.125)
    close(got, ref.attend(pool, table, q, seq, pos, heads, 0.125))


def device_pool(shape, n_seq, ctx, page, seed=0):
    """A cache filled on the GPU by store(): for contexts too long for the
    reference.  Returns (cache, keys, values as stored [seq, ctx, n_kv, d] f64)."""
    import torch

    from moe_amd.paged import KvCache

    heads, n_kv, qd, vd = shape
    mp = -(-ctx // page)
    g = torch.Generator(device="cuda").manual_seed(seed)
    table = torch.randperm(n_seq * mp, generator=g, device="cuda").to(torch.int32).view(n_seq, mp)
    cache = KvCache.new(n_seq * mp, table, n_kv=n_kv, qd=qd, vd=vd, page=page, means=True)
    slots = (table.long()[:, :, None] * page + torch.arange(page, device="cuda")).view(-1)
    k, v = (torch.randn((len(slots), n_kv * d), generator=g, device="cuda") for d in (qd, vd))
    cache.store(k, v, slots)
    kb, vb = torch.empty_like(k), torch.empty_like(v)
    cache.load(slots, kb, vb)
    return cache, kb.view(n_seq, mp * page, n_kv, qd).double(), vb.view(n_seq, mp * page, n_kv, vd).double()


def attend64(k, v, q, seq, pos, heads, scale, window=0):
    import torch

    n_kv = k.shape[2]
    rep = heads // n_kv
    out = []
    for r, (s, p) in enumerate(zip(seq, pos)):
        lo = max(0, p + 1 - window) if window else 0
        qq = q[r].double().view(n_kv, rep, -1)
        w = torch.softmax(torch.einsum("ghd,pgd->ghp", qq, k[s, lo:p + 1]) * scale, -1)
        out.append(torch.einsum("ghp,pgd->ghd", w, v[s, lo:p + 1]).reshape(-1))
    return torch.stack(out).cpu().numpy()


@pytest.mark.parametrize("shape,ctx,rows", [
    ((32, 8, 128, 128), 40000, [(0, 39999)]),
    ((16, 16, 192, 128), 9000, [(0, 8999), (0, 4500)]),
    ((8, 2, 64, 64), 30000, [(0, p) for p in range(29990, 30000)]),
    ((4, 2, 256, 256), 20001, [(0, 20000)]),
    ((32, 8, 128, 128), 3000, [(0, p) for p in range(2500, 3000)]),
    ((32, 32, 128, 128), 900, [(0, p) for p in range(900)]),
    ((32, 8, 128, 128), 2000, [(0, p) for p in range(700, 2000)]),
])
def test_long_contexts_and_prompts(shape, ctx, rows):
    """One sequence far along (its positions go to many blocks), and long runs
    of rows (many blocks of rows); loosely bounded positions change nothing."""
    import torch

    heads, n_kv, qd, vd = shape
    cache, k, v = device_pool(shape, 1, ctx, 64)
    seq, pos = zip(*rows)
    q = torch.randn((len(rows), heads * qd), generator=torch.Generator(device="cuda").manual_seed(7), device="cuda") * 2
    pick = list(range(0, len(rows), max(1, len(rows) // 40)))
    for window in (0, 700):
        for bound in (max(pos), cache.table.shape[1] * 64 - 1):
            got = run_attend(cache, q.cpu().numpy(), seq, pos, heads, qd ** -0.5, window, max_pos=bound)
            want = attend64(k, v, q[pick], [seq[i] for i in pick], [pos[i] for i in pick], heads, qd ** -0.5, window)
            # Scores twice those of the other tests.
            close(got[pick], want, 2 * TOL)


@pytest.mark.parametrize("shape,rows", [((16, 2, 64, 64), 5), ((16, 2, 64, 64), 1024), ((32, 8, 128, 128), 1100)], ids=str)
def test_positions_past_2_30(shape, rows):
    """A sequence of more than 2^30 positions, a page in the middle of the
    window missing: few rows, and enough of them for the wide groups."""
    import torch

    from moe_amd.paged import KvCache

    heads, n_kv, d, _ = shape
    page, mid = 4096, 1 << 18
    few, k, v = device_pool(shape, 1, 2 * page, page)
    table = torch.full((1, mid + 1), -1, dtype=torch.int32, device="cuda")
    table[0, mid - 2], table[0, mid] = few.table[0, 0], few.table[0, 1]
    cache = KvCache(few.pool, table, n_kv=n_kv, qd=d, vd=d, page=page)
    q = torch.randn((rows, heads * d), generator=torch.Generator(device="cuda").manual_seed(1), device="cuda")
    got = run_attend(cache, q.cpu().numpy(), [0] * rows, [mid * page + r for r in range(rows)], heads, 0.125, 2 * page)
    pick = list(range(0, rows, max(1, rows // 20)))
    # without the missing page the rows are at 4096 + r, with a window of 4096
    close(got[pick], attend64(k, v, q[pick], [0] * len(pick), [page + r for r in pick], heads, 0.125, page))


@pytest.mark.parametrize("shape,rows", [((8, 2, 64, 64), 3), ((6, 2, 96, 96), 40), ((16, 2, 64, 64), 1024), ((16, 2, 96, 64), 1024),
                                        ((32, 8, 128, 128), 1100)], ids=str)
def test_unseen_sizes_do_not_matter(shape, rows):
    """Values 10^11 times those that the rows see, before their window and in
    the rest of the last page: outputs keep their relative precision."""
    import torch

    heads, n_kv, qd, vd = shape
    first, window, page = 100, 45, 64
    cache, k, v = device_pool(shape, 1, first + rows + 60, page)
    top = first + rows - 1
    h = torch.rand((cache.table.shape[1] * page, n_kv, vd // 32), generator=torch.Generator(device="cuda").manual_seed(2),
                   device="cuda")
    size = torch.full_like(h, 6e-7)  # f16 subnormals
    size[:first + 1 - window] = 6e4
    size[top + 1:] = 6e4
    scale = ((0.5 + 0.5 * h) * size).half()
    # Into the tiles: number 32 b + 8 (p % 16 / 4) + 4 (p / 16) + p % 4 of the region, page by page.
    tiles = cache.pool.view(-1, n_kv, page // 32, 18 * (qd + vd))
    p = torch.arange(32, device="cuda")
    at = 8 * (p % 16 // 4) + 4 * (p // 16) + p % 4
    new = torch.empty((len(tiles), n_kv, page // 32, vd // 32, 32), dtype=torch.float16, device="cuda")
    new[cache.table[0].long()] = scale.view(-1, page // 32, 32, n_kv, vd // 32).permute(0, 3, 1, 4, 2)[..., at.argsort()]
    tiles[..., 18 * qd + 16 * vd:] = new.view(*new.shape[:3], -1).view(torch.uint8)
    slots = (cache.table[0].long()[:, None] * page + torch.arange(page, device="cuda")).view(-1)
    kb, vb = torch.empty((len(slots), n_kv * qd), device="cuda"), torch.empty((len(slots), n_kv * vd), device="cuda")
    cache.load(slots, kb, vb)
    assert vb[first + 1 - window:top + 1].abs().max() < 1e-5 and vb[top + 1:].abs().max() > 1e5
    q = torch.randn((rows, heads * qd), generator=torch.Generator(device="cuda").manual_seed(1), device="cuda")
    got = run_attend(cache, q.cpu().numpy(), [0] * rows, [first + r for r in range(rows)], heads, qd ** -0.5, window)
    pick = list(range(0, rows, max(1, rows // 20)))
    close(got[pick], attend64(kb.view(1, -1, n_kv, qd).double(), vb.view(1, -1, n_kv, vd).double(), q[pick], [0] * len(pick),
                              [first + r for r in pick], heads, qd ** -0.5, window))


def blocks_close(got, cache, table_slots, q, seq, pos, heads, scale, tol, window=0, lists=None):
    """Per row, head and 32-value block: the largest error against the largest
    of the block's sums of |weight value|, which is what f32 sums are off by a
    share of.  The cache's values as they read back, in 64 bits."""
    import torch

    n_seq, ctx = table_slots.shape
    n_kv, qd, vd, rep = cache.n_kv, cache.qd, cache.vd, heads // cache.n_kv
    kb, vb = (torch.empty((n_seq * ctx, n_kv * d), device="cuda") for d in (qd, vd))
    cache.load(table_slots.reshape(-1), kb, vb)
    k, v = kb.view(n_seq, ctx, n_kv, qd).double(), vb.view(n_seq, ctx, n_kv, vd).double()
    errors = []
    for r, (s, p) in enumerate(zip(seq, pos)):
        lo = max(0, p + 1 - window) if window else 0
        qq = q[r].double().view(n_kv, rep, qd)
        kk, vv = (x[s, lo:p + 1].permute(1, 0, 2).contiguous() for x in (k, v))
        score = torch.matmul(qq, kk.transpose(1, 2).contiguous()) * scale
        if lists is not None:  # [row, kv head, page]: whether it is listed
            score.masked_fill_(~lists[r][:, torch.arange(lo, p + 1, device="cuda") // cache.page][:, None], -math.inf)
        w = torch.softmax(score, -1)
        want, size = torch.matmul(w, vv).view(heads, -1, 32), torch.matmul(w, vv.abs()).view(heads, -1, 32).amax(-1)
        err = (torch.from_numpy(got[r]).cuda().double().view(heads, -1, 32) - want).abs().amax(-1)
        assert bool(torch.isfinite(size).all()) and bool((err[size == 0] == 0).all())
        errors.append(float((err / size.clamp(min=1e-300)).max()))
    assert np.max(errors) < tol, np.max(errors)  # (a NaN is none)


UNEVEN = {  # shape, positions, rows
    "one_row": ((8, 2, 64, 64), 200, [190]), "rows": ((8, 2, 64, 64), 200, range(150, 190)),
    "latent": ((16, 16, 192, 128), 150, range(130, 140)), "96": ((6, 2, 96, 96), 150, range(100, 140)),
    "224": ((1, 1, 224, 64), 100, [60, 99]), "256": ((4, 2, 256, 256), 100, range(80, 90)),
    "parts": ((32, 8, 128, 128), 9000, [8990]), "prompt": ((32, 8, 128, 128), 1200, range(20, 1200)),
    "wide": ((32, 32, 128, 128), 1200, range(60, 1200))}


@pytest.mark.parametrize("how", ["block", "early", "late", "silent", "mixed", "subnormal"])
@pytest.mark.parametrize("name", list(UNEVEN))
def test_uneven_values_keep_their_precision(name, how):
    """What is small among a head's values is as exact as if it were alone:
    one block of 32 dims 2^-16 of the others (or a subnormal scale's size); a
    position whose values are 2^20 times the others' and that hardly weighs
    anything, before or behind them; one that takes nearly all weight and is 0;
    every block of a size of its own.

    Tolerance: sums of up to 9000 products in f32, sqrt(9000) 2^-24 and 2^-22
    of the two pieces, are within TOL.  A score S is off by 2^-22 S (the query's
    two pieces) and 2^-24 S (its sum in f32), and a weight by as much; scores
    that weigh are below 6 but for the silent position's 13."""
    import torch

    from moe_amd.paged import KvCache

    (heads, n_kv, qd, vd), ctx, rows = UNEVEN[name]
    page = 64
    mp = -(-ctx // page)
    g = torch.Generator(device="cuda").manual_seed(len(name))
    table = torch.randperm(mp, generator=g, device="cuda").to(torch.int32).view(1, mp)
    cache = KvCache.new(mp, table, n_kv=n_kv, qd=qd, vd=vd, page=page)
    slots = (table.long()[:, :, None] * page + torch.arange(page, device="cuda")).view(1, -1)
    k = torch.randn((mp * page, n_kv, qd), generator=g, device="cuda")
    v = torch.randn((mp * page, n_kv, vd), generator=g, device="cuda")
    q = torch.randn((len(rows), heads, qd), generator=g, device="cuda")
    scale, S = qd ** -0.5, 6.0
    q[..., 0], k[..., 0] = 2.0, 0.0
    at = {"early": 3, "late": min(rows) - 2, "silent": 0}.get(how)
    if how == "block":
        v[..., -32:] *= 2.0 ** -16
    elif how == "subnormal":
        v[..., :32] *= 2.0 ** -18
    elif how == "mixed":
        v *= torch.exp2(torch.randint(-11, 12, (mp * page, n_kv, vd // 32, 1), generator=g, device="cuda").float()) \
            .expand(-1, -1, -1, 32).reshape(v.shape)
    else:
        k[at], q[..., 1:32] = 0.0, 0.0
        k[at, :, 0] = (13.0 if how == "silent" else -28.0) / scale / 2.0
        v *= 2.0 ** -8
        v[at] *= 0.0 if how == "silent" else 2.0 ** 20
        S = 13.0
    cache.store(k.view(len(k), -1), v.view(len(v), -1), slots.view(-1))
    got = run_attend(cache, q.view(len(rows), -1).cpu().numpy(), [0] * len(rows), list(rows), heads, scale)
    pick = list(range(0, len(rows), max(1, len(rows) // 25)))
    blocks_close(got[pick], cache, slots, q.view(len(rows), -1)[pick], [0] * len(pick), [rows[i] for i in pick], heads, scale,
                 TOL + S * (2.0 ** -22 + 2.0 ** -24))


@pytest.mark.parametrize("shape", [(8, 2, 64, 64), (16, 16, 192, 128), (32, 8, 128, 128), (6, 2, 96, 96)], ids=str)
@pytest.mark.parametrize("window", [0, 45, 2 ** 31 - 1])
def test_uneven_values_in_windows_and_lists(shape, window):
    """Every block of a size of its own, 2^22 between them, read through a
    window, or through lists of pages that differ from row to row."""
    import torch

    from moe_amd.paged import KvCache

    heads, n_kv, qd, vd = shape
    ctx, page = 400, 32
    mp = -(-ctx // page)
    g = torch.Generator(device="cuda").manual_seed(3)
    table = torch.randperm(mp, generator=g, device="cuda").to(torch.int32).view(1, mp)
    cache = KvCache.new(mp, table, n_kv=n_kv, qd=qd, vd=vd, page=page)
    slots = (table.long()[:, :, None] * page + torch.arange(page, device="cuda")).view(1, -1)
    size = torch.exp2(torch.randint(-11, 12, (mp * page, n_kv * vd // 32, 1), generator=g, device="cuda").float())
    v = (torch.randn((mp * page, n_kv * vd // 32, 32), generator=g, device="cuda") * size).view(mp * page, -1)
    cache.store(torch.randn((mp * page, n_kv * qd), generator=g, device="cuda"), v, slots.view(-1))
    rows = list(range(130, 400, 7))
    q = torch.randn((len(rows), heads * qd), generator=g, device="cuda")
    listed = torch.rand((len(rows), n_kv, mp), generator=g, device="cuda") < 0.4
    listed[..., 0] = True
    lists = torch.full((len(rows), n_kv, mp), -1, dtype=torch.int32, device="cuda")
    at = torch.where(listed, torch.arange(mp, device="cuda"), mp).sort(-1).values
    lists.copy_(torch.where(at < mp, at, -1))
    # scores below 6, as above
    tol = TOL + 6 * (2.0 ** -22 + 2.0 ** -24)
    got = run_attend(cache, q.cpu().numpy(), [0] * len(rows), rows, heads, qd ** -0.5, window)
    blocks_close(got, cache, slots, q, [0] * len(rows), rows, heads, qd ** -0.5, tol, window)
    if window != 45:  # (a row's pages might all lie before it)
        got = run_attend(cache, q.cpu().numpy(), [0] * len(rows), rows, heads, qd ** -0.5, window, lists.cpu().numpy())
        blocks_close(got, cache, slots, q, [0] * len(rows), rows, heads, qd ** -0.5, tol, window, listed)


@pytest.mark.parametrize("used", [3, 40, 700])
def test_room_for_more_rows_than_there_are(used):
    """A captured step has room for many rows, of which most are none: so many
    that groups of 64 columns are formed around a few sequences that decode."""
    import torch

    shape, room = (32, 8, 128, 128), 1500
    heads, n_kv, d, _ = shape
    cache, k, v = device_pool(shape, 40, 320, 64)
    rows = [(i % 40, 319 - i % 90) for i in range(min(used, 40))] + [(7, p) for p in range(used - 40)][:320]
    rows += [(3, p) for p in range(used - len(rows))][:320]
    assert max(p for _, p in rows) < 320
    seq, pos = zip(*(rows + [(-1, -1)] * (room - len(rows))))
    q = torch.randn((room, heads * d), generator=torch.Generator(device="cuda").manual_seed(7), device="cuda")
    out = torch.full((room, heads * d), 7.0, device="cuda")
    args = q, ints(seq), ints(pos), out
    call = lambda: cache.attend(*args, max_pos=cache.table.shape[1] * 64 - 1, scale=d ** -0.5)  # noqa: E731
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for _ in range(3):
        out.fill_(7.0)
        q.normal_(generator=torch.Generator(device="cuda").manual_seed(9))
        graph.replay()
        torch.cuda.synchronize()
        got = out.cpu().numpy()
        assert (got[len(rows):] == 7.0).all()
        pick = list(range(0, len(rows), max(1, len(rows) // 60)))
        close(got[pick], attend64(k, v, q[pick], [seq[i] for i in pick], [pos[i] for i in pick], heads, d ** -0.5))


@pytest.mark.parametrize("window", [0, 90])
@pytest.mark.parametrize("shape", [(100, 1, 64, 64), (96, 2, 96, 32), (32, 8, 128, 128), (16, 16, 192, 128), (90, 3, 224, 64),
                                   (128, 8, 128, 128), (100, 1, 128, 128)], ids=str)
def test_ragged_batches_of_many_rows(shape, window):
    """Sequences of different lengths, rows that are none between them, rows in
    no order, more query heads a kv head than a block's columns."""
    import torch

    heads, n_kv, qd, vd = shape
    cache, k, v = device_pool(shape, 5, 700, 64)
    g = np.random.default_rng(0)
    rows = ([(0, p) for p in range(299)] + [(0, -1)] * 3 + [(3, p) for p in range(651, 700)] + [(7, 20)] * 5 +
            [(1, p) for p in range(5, 250)] + [(-1, 9)] + [(2, int(p)) for p in g.integers(0, 700, 50)] + [(4, 699)])
    seq, pos = zip(*rows)
    q = torch.randn((len(rows), heads * qd), generator=torch.Generator(device="cuda").manual_seed(7), device="cuda")
    got = run_attend(cache, q.cpu().numpy(), seq, pos, heads, qd ** -0.5, window)
    none = [i for i, (a, p) in enumerate(rows) if p < 0 or not 0 <= a < 5]
    assert (got[none] == 7.0).all()
    pick = [i for i in range(len(rows)) if i not in none and (i % 9 == 0 or i > len(rows) - 40)]
    close(got[pick], attend64(k, v, q[pick], [seq[i] for i in pick], [pos[i] for i in pick], heads, qd ** -0.5, window))


@pytest.mark.parametrize("window", [0, 70])
@pytest.mark.parametrize("shape", [(32, 8, 128, 128), (32, 32, 128, 128), (21, 3, 128, 128), (36, 3, 128, 128), (40, 2, 128, 128),
                                   (64, 2, 128, 128), (80, 1, 128, 128)], ids=str)
def test_wide_groups_of_mixed_rows(shape, window):
    """So many rows that groups of 64 columns are formed, of which some are one
    run (prompts), some several (sequences that decode, a prompt's end, rows that
    are none), some one of few columns: 1 to 80 query heads a kv head."""
    heads, n_kv, d, _ = shape
    n_seq = 40
    cache, k, v = device_pool(shape, n_seq, 200, 64)
    g = np.random.default_rng(1)
    # enough for 512 groups of 64 columns
    rows, want = [], 512 // n_kv * 64 // (heads // n_kv) + 70
    for i in range(n_seq):
        rows += [(i, int(g.integers(0, 200)))]
    rows += [(0, -1)] * 70 + [(5, 199)] + [(-1, 3)] * 70
    while len(rows) < want:
        n, s = int(g.integers(2, 200)), int(g.integers(0, n_seq))
        rows += [(s, p) for p in range(200 - n, 200)]
        rows += [(int(g.integers(0, n_seq)), int(g.integers(0, 200))) for _ in range(int(g.integers(0, 20)))]
    seq, pos = zip(*rows)
    import torch

    q = torch.randn((len(rows), heads * d), generator=torch.Generator(device="cuda").manual_seed(7), device="cuda")
    got = run_attend(cache, q.cpu().numpy(), seq, pos, heads, d ** -0.5, window)
    none = [i for i, (a, p) in enumerate(rows) if p < 0 or not 0 <= a < n_seq]
    assert (got[none] == 7.0).all()
    there = [i for i in range(len(rows)) if i not in set(none)]
    pick = there[:60] + there[60::max(1, len(there) // 300)] + there[-20:]
    close(got[pick], attend64(k, v, q[pick], [seq[i] for i in pick], [pos[i] for i in pick], heads, d ** -0.5, window))
    # and each row as it is in a call of few rows
    few = pick[::40]
    part = run_attend(cache, q[few].cpu().numpy(), [seq[i] for i in few], [pos[i] for i in few], heads, d ** -0.5, window)
    close(part, got[few])


def test_many_sequences_cost_what_their_halves_do():
    """A decode step of 1024 sequences in one call, against two calls of 512,
    each the shortest of several: groups of 64 columns are for runs that fill
    them (in such groups the one call took 2.5 times the two)."""
    import torch

    heads, n_kv, d, n, ctx = 32, 8, 128, 1024, 320
    cache, _, _ = device_pool((heads, n_kv, d, d), n, ctx, 64)
    q = torch.randn((n, heads * d), device="cuda")
    out = torch.empty_like(q)
    seq, pos = ints(range(n)), ints([ctx - 1 - i % 50 for i in range(n)])

    def time_of(*parts):
        best = 1e9
        for _ in range(8):
            a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
            a.record()
            for _ in range(4):
                for lo, hi in parts:
                    cache.attend(q[lo:hi], seq[lo:hi], pos[lo:hi], out[lo:hi], max_pos=ctx - 1, scale=d ** -0.5)
            b.record()
            torch.cuda.synchronize()
            best = min(best, a.elapsed_time(b))
        return best

    assert time_of((0, n)) < 1.5 * time_of((0, n // 2), (n // 2, n))


def test_load_of_keys_or_values_alone():
    import torch

    cache, k, v = device_pool((6, 3, 96, 160), 1, 100, 32)
    slots = torch.tensor([5, -1, 70, 31, 10 ** 9], device="cuda")
    whole = [torch.full((5, 3 * d), 7.0, device="cuda") for d in (96, 160)]
    cache.load(slots, *whole)
    for i in range(2):
        one = torch.full_like(whole[i], 7.0)
        cache.load(slots, *((one, None) if i == 0 else (None, one)))
        assert torch.equal(one, whole[i]) and (one[[1, 4]] == 7.0).all() and (one[0] != 7.0).any()
    cache.load(slots)


def test_a_pool_past_4_gib():
    """Pages whose bytes, and rows' slots, lie past 32 bits: written, read,
    attended to and chosen as the same rows are in a small pool."""
    import torch

    from moe_amd.paged import KvCache

    heads, n_kv, d, page, ctx = 32, 8, 128, 64, 1000
    near, k, v = device_pool((heads, n_kv, d, d), 1, ctx, page)
    mp = near.table.shape[1]
    n_pages = (5 << 30) // KvCache.page_bytes(n_kv, d, d, page)
    table = (n_pages - 1 - torch.arange(mp, dtype=torch.int32, device="cuda")).view(1, mp)
    far = KvCache.new(n_pages, table, n_kv=n_kv, qd=d, vd=d, page=page, means=True)
    slot = lambda c: (c.table[0].long()[:, None] * page + torch.arange(page, device="cuda")).view(-1)  # noqa: E731
    kv = [torch.randn((mp * page, n_kv * d), generator=torch.Generator(device="cuda").manual_seed(i), device="cuda")
          for i in range(2)]
    q = torch.randn((3, heads * d), generator=torch.Generator(device="cuda").manual_seed(5), device="cuda")
    seq, pos = ints([0] * 3), ints([999, 700, 998])
    got = []
    for c in (near, far):
        c.store(*kv, slot(c))
        back = [torch.empty_like(x) for x in kv]
        c.load(slot(c), *back)
        lists, out = torch.empty((3, n_kv, 5), dtype=torch.int32, device="cuda"), torch.empty_like(q)
        c.select(q, seq, pos, lists, max_pos=999)
        c.attend(q, seq, pos, out, max_pos=999, scale=d ** -0.5, pages=lists)
        got.append([*back, lists, out])
    for a, b in zip(*got):
        assert torch.equal(a, b)


# ------------------------------------------------------------- choice of pages


@pytest.mark.parametrize("shape", [(8, 2, 64, 64), (16, 16, 192, 128), (32, 8, 128, 128), (6, 2, 96, 96), (40, 1, 64, 32)],
                         ids=str)
@pytest.mark.parametrize("n_seq,mp,n_sel,sinks,recent", [(3, 1, 1, 0, 1), (4, 40, 5, 1, 2), (2, 300, 16, 0, 1),
                                                        (1, 1500, 64, 2, 3), (2, 20, 30, 1, 1)])
def test_select(shape, n_seq, mp, n_sel, sinks, recent):
    import torch

    heads, n_kv, qd, vd = shape
    page = 32
    g = np.random.default_rng(mp)
    n_pages = n_seq * mp + 2
    table = g.permutation(n_pages)[:n_seq * mp].reshape(n_seq, mp).astype(np.int32)
    means = g.standard_normal((n_pages, n_kv, qd)).astype(np.float16)
    if mp >= 20:
        means[table[0, 3]] = means[table[0, 9]] = means[table[0, 5]]  # equal scores: the lower page
        means[table[0, 7]], means[table[0, 8], :, 3], means[table[0, 6], :, 0] = np.nan, np.inf, -np.inf
        table[0, 11] = n_pages
    rows = [(s, int(p)) for s in range(n_seq) for p in (0, page - 1, min(page, mp * page - 1), mp * page - 1, mp * page // 2)]
    rows += [(0, -1), (-1, 5), (n_seq, 5)]
    seq, pos = zip(*rows)
    q = g.standard_normal((len(rows), heads * qd)).astype(np.float32)
    pool = torch.zeros(n_pages * n_kv * 18 * (qd + vd), dtype=torch.uint8, device="cuda")
    from moe_amd.paged import KvCache

    cache = KvCache(pool, torch.from_numpy(table).cuda(), n_kv=n_kv, qd=qd, vd=vd, page=page, means=torch.from_numpy(means).cuda())
    lists = torch.full((len(rows), n_kv, n_sel), 77, dtype=torch.int32, device="cuda")
    want = ref.select(means, table, q, seq, pos, heads, page, n_sel, sinks, recent)
    for bound in (max(pos), mp * page - 1):
        cache.select(torch.from_numpy(q).cuda(), ints(seq), ints(pos), lists, max_pos=bound, sinks=sinks, recent=recent)
        assert np.array_equal(lists.cpu().numpy(), want)


@pytest.mark.parametrize("n_seq,mp,n_sel", [(1, 5000, 20), (40, 700, 33), (9, 4097, 256)])
def test_select_many_pages(n_seq, mp, n_sel):
    """Scores through the workspace, and in LDS up to its end; few distinct
    scores, so that the last one chosen is one of many equal ones."""
    import torch

    from moe_amd.paged import KvCache

    heads, n_kv, d, page = 2, 2, 32, 32
    g = torch.Generator(device="cuda").manual_seed(mp)
    table = torch.randperm(n_seq * mp, generator=g, device="cuda").to(torch.int32).view(n_seq, mp)
    means = torch.randint(-2, 3, (n_seq * mp, n_kv, 1), generator=g, device="cuda").half().expand(-1, -1, d).contiguous()
    pool = torch.zeros(n_seq * mp * n_kv * 18 * 2 * d, dtype=torch.uint8, device="cuda")
    cache = KvCache(pool, table, n_kv=n_kv, qd=d, vd=d, page=page, means=means)
    q = torch.ones((n_seq, heads * d), device="cuda")
    seq, pos = ints(range(n_seq)), ints([mp * page - 1 - 40 * i for i in range(n_seq)])
    lists = torch.empty((n_seq, n_kv, n_sel), dtype=torch.int32, device="cuda")
    cache.select(q, seq, pos, lists, max_pos=mp * page - 1, sinks=1, recent=2)
    got = lists.cpu().numpy()
    score = means[table.long()].double().sum(-1).cpu().numpy()  # [seq, page, kv]
    for s in range(n_seq):
        cur = int(pos[s]) // page
        for kv in range(n_kv):
            x = score[s, :cur + 1, kv].copy()
            x[0] = x[cur - 1:] = np.inf
            assert got[s, kv].tolist() == sorted(np.argsort(-x, kind="stable")[:n_sel].tolist())


@pytest.mark.parametrize("size,spread", [(1.0, 0.0), (1e-30, 0.0), (1e25, 0.0), (1.0, 20.0)])
@pytest.mark.parametrize("near", [2, 40, 200, 500])
@pytest.mark.parametrize("shape", [(32, 8, 128, 128), (6, 2, 96, 96), (40, 2, 64, 32), (4, 2, 256, 256), (8, 2, 192, 128)], ids=str)
def test_select_near_scores(shape, near, size, spread):
    """Pages whose scores differ by less than f32 sums resolve around the last
    one chosen, few of them and more than are settled together; mean keys among
    f16's subnormals; queries of any size, heads e^20 apart."""
    import torch

    from moe_amd.paged import KvCache

    heads, n_kv, qd, vd = shape
    page, mp, n_sel, n_seq = 32, 600, 20, 3
    g = np.random.default_rng(near)
    means = (g.standard_normal((n_seq * mp, n_kv, qd)) * np.array([1, 6e-6, 1e4]).repeat(mp)[:, None, None]).astype(np.float16)
    table = np.stack([g.permutation(mp) + s * mp for s in range(n_seq)]).astype(np.int32)
    q = (g.standard_normal((n_seq, heads, qd)) * size * np.exp(spread * g.standard_normal((n_seq, heads, 1)))).astype(np.float32)
    for s in range(n_seq):
        at = g.permutation(np.arange(5, mp - 5))[:near]
        top = means[table[s, at[0]]]
        for kv in range(n_kv):  # along the first head: well above the others
            qq = q[s, kv * (heads // n_kv)]
            top[kv] = (qq / np.abs(qq).max() * 4 * np.array([1, 6e-6, 1e4])[s]).astype(np.float16)
        bits = np.broadcast_to(top.view(np.uint16), (near, n_kv, qd)).copy()
        bits[np.arange(near), :, g.integers(0, qd, near)] += g.integers(0, 2, (near, 1), dtype=np.uint16)
        means[table[s, at]] = bits.view(np.float16)
    pool = torch.zeros(len(means) * n_kv * 18 * (qd + vd), dtype=torch.uint8, device="cuda")
    d = lambda x: torch.from_numpy(x).cuda()  # noqa: E731
    cache = KvCache(pool, d(table), n_kv=n_kv, qd=qd, vd=vd, page=page, means=d(means))
    pos = [mp * page - 1, mp * page - 40, mp * page - 1]
    lists = torch.empty((n_seq, n_kv, n_sel), dtype=torch.int32, device="cuda")
    cache.select(d(q.reshape(n_seq, -1)), ints(range(n_seq)), ints(pos), lists, max_pos=mp * page - 1, sinks=1, recent=2)
    got = lists.cpu().numpy()
    for s in range(n_seq):
        cur = pos[s] // page
        for kv in range(n_kv):
            qq = q[s].reshape(n_kv, -1, qd)[kv].astype(np.float64)
            x = (means[table[s, :cur + 1], kv].astype(np.float64) @ qq.T).max(-1)
            x[0] = x[cur - 1:] = np.inf
            assert got[s, kv].tolist() == sorted(np.argsort(-x, kind="stable")[:n_sel].tolist())


# ------------------------------------------- calls together, streams and graphs


def one_step(cache, table, rows, add, k, v, q, out, lists, max_pos, scale):
    table.advance(add, rows)
    cache.store(k, v, rows.slot)
    cache.select(q, rows.seq, rows.pos, lists, max_pos=max_pos, sinks=1, recent=1)
    cache.attend(q, rows.seq, rows.pos, out[0], max_pos=max_pos, scale=scale)
    cache.attend(q, rows.seq, rows.pos, out[1], max_pos=max_pos, scale=scale, pages=lists)


@pytest.mark.parametrize("how", ["eager", "stream", "graph"])
def test_steps_together(how):
    """Tables, cache write, page choice, dense and sparse attention as a decode
    loop runs them: sequences of differing lengths grow and end, against the
    plain forms step by step; the same from a captured step, replayed."""
    import torch

    from moe_amd.paged import KvCache, PageTable, Rows

    n, page, mp, n_pages, heads, n_kv, d, n_sel, room = 5, 32, 8, 30, 8, 2, 64, 3, 40
    g = np.random.default_rng(11)
    table = PageTable.new(n, mp, n_pages, page, "cuda")
    cache = KvCache.new(n_pages, table.table, n_kv=n_kv, qd=d, vd=d, page=page, means=True)
    rows = Rows.new(n, room, "cuda")
    add = torch.zeros(n, dtype=torch.int32, device="cuda")
    k, v = torch.zeros((room, n_kv * d), device="cuda"), torch.zeros((room, n_kv * d), device="cuda")
    q, out = torch.zeros((room, heads * d), device="cuda"), torch.zeros((2, room, heads * d), device="cuda")
    lists = torch.zeros((room, n_kv, n_sel), dtype=torch.int32, device="cuda")
    args = (cache, table, rows, add, k, v, q, out, lists, mp * page - 1, d ** -0.5)
    graph = None
    if how == "graph":
        one_step(*args)  # adds nothing
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            one_step(*args)
    side = torch.cuda.Stream()
    pool = ref.Pool(n_pages, n_kv, d, d, page)
    length, state = np.zeros(n, np.int32), np.array([0, n_pages], np.int32)
    tab, ring = np.full((n, mp), -1, np.int32), np.arange(n_pages, dtype=np.int32)
    means = np.zeros((n_pages, n_kv, d), np.float16)
    for step in range(40):
        a = np.ones(n, np.int32) if step % 7 else g.integers(0, 9, n).astype(np.int32)
        if step % 11 == 10:
            a[int(g.integers(0, n))] = -1
        if step % 13 == 0:
            a[1] = 30
        new = [g.standard_normal(x.shape).astype(np.float32) for x in (k, v, q)]
        for x, y in zip((k, v, q), new):
            x.copy_(torch.from_numpy(y))
        add.copy_(torch.from_numpy(a))
        out.fill_(3.0)
        if how == "graph":
            graph.replay()
        elif how == "stream":
            torch.cuda.synchronize()
            with torch.cuda.stream(side):
                one_step(*args)
            side.synchronize()
        else:
            one_step(*args)
        torch.cuda.synchronize()
        w = ref.advance(length, a, tab, ring, state, page, room)
        length, state = w["length"], w["state"]
        assert rows.slot.cpu().numpy().tolist() == w["slot"] and rows.status.cpu().numpy().tolist() == w["status"]
        pool.store(w["slot"], new[0], new[1])
        assert np.array_equal(cache.pool.cpu().numpy(), pool.raw)
        for s in w["slot"]:
            if s >= 0 and s % page == page - 1:
                means[s // page] = pool.mean(s // page)
        assert np.array_equal(cache.means.cpu().numpy(), means)
        want = ref.select(means, tab, new[2], w["seq"], w["pos"], heads, page, n_sel, 1, 1)
        assert np.array_equal(lists.cpu().numpy(), want)
        for i, some in enumerate((None, want)):
            close(out[i].cpu().numpy(), ref.attend(pool, tab, new[2], w["seq"], w["pos"], heads, d ** -0.5, 0, some,
                                                   np.full((room, heads * d), 3.0)))


def test_calls_on_a_stream_that_is_not_current():
    """stream= another one: the scratch of two calls at once is each one's own."""
    import torch

    shape = (32, 8, 128, 128)
    cache, k, v = device_pool(shape, 1, 20000, 64)
    q = torch.randn((2, 32 * 128), device="cuda")
    seq, pos = ints([0]), ints([19990])
    want = attend64(k, v, q, [0, 0], [19990, 19990], 32, 128 ** -0.5)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = [torch.zeros((1, 32 * 128), device="cuda") for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(20):
        for i in range(2):
            cache.attend(q[i:i + 1], seq, pos, outs[i], max_pos=19990, scale=128 ** -0.5,
                         stream=streams[i] if i else streams[i].cuda_stream)
    torch.cuda.synchronize()
    for i in range(2):
        close(outs[i].cpu().numpy(), want[i:i + 1])


def test_two_graphs_replayed_at_once():
    """Two captured attentions keep scratch of their own."""
    import torch

    shape = (32, 8, 128, 128)
    cache, k, v = device_pool(shape, 1, 20000, 64)
    seq, pos = ints([0]), ints([19990])
    graphs, qs, outs = [], [], []
    for i in range(2):
        q, out = torch.randn((1, 32 * 128), device="cuda"), torch.zeros((1, 32 * 128), device="cuda")
        call = lambda: cache.attend(q, seq, pos, out, max_pos=19990, scale=128 ** -0.5)  # noqa: E731
        call()
        torch.cuda.synchronize()
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            call()
        graphs.append(gr)
        qs.append(q)
        outs.append(out)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for rep in range(3):
        for i in range(2):
            qs[i].normal_()
        torch.cuda.synchronize()
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                graphs[i].replay()
        torch.cuda.synchronize()
        for i in range(2):
            close(outs[i].cpu().numpy(), attend64(k, v, qs[i], [0], [19990], 32, 128 ** -0.5))
