"""The paged 8-bit cache on the GPU (moe_kv8_*) against the plain 64-bit forms
of kv8_reference.py.

Codes and scales are defined with every step rounded to f32, so stored bytes
are compared for equality.

Tolerance of attention.  A score's error: the query in 24-bit pieces, half a
step of 2^-22 of the head's largest at most, over qd products added up in whole
numbers (about sqrt(qd) 2^-23 of their terms' size), and the f32 roundings of
its scales (3 x 2^-24 of itself); for the scores of order 1 here that is below
2e-6 of the weight.  Weights are held to 2^-21 of the largest product of weight
and scale and summed in f32.  gpu_util.TOL = 5e-6 of the largest output is the
bar of moe_attention on the same quantities.  Larger scores carry larger errors
in proportion; the tests that make them say so."""
import numpy as np
import pytest

import kv8_reference as ref
from gpu_util import TOL

pytestmark = pytest.mark.gpu

HEADS = [(8, 2, 64, 64), (16, 16, 192, 128), (32, 8, 128, 128), (6, 2, 96, 96), (40, 1, 64, 32), (4, 2, 256, 256),
         (3, 3, 32, 160), (48, 2, 128, 128), (1, 1, 224, 64)]
# name: (sequence, position) of each row
ROWS = {
    "decode": [(s, p) for s, p in enumerate([0, 15, 16, 63, 64, 65, 130, 127, 128, 1, 299])],
    "one_row": [(0, 200)],
    "first": [(0, 0)],
    "prompt": [(0, p) for p in range(37)],
    "chunk": [(0, 100 + p) for p in range(70)],
    "mixed": [(0, p) for p in range(9)] + [(1, 40 + p) for p in range(21)] + [(2, 5), (3, 77)] +
             [(0, 9 + p) for p in range(13)] + [(1, -1), (-1, 3), (11, 3)],
    "shuffled": [(0, p) for p in (90, 3, 50, 51, 7, 0, 128)],
}


def cuda(x):
    import torch

    return torch.from_numpy(np.ascontiguousarray(x)).cuda()


def ints(v, t="int32"):
    import torch

    return torch.tensor([int(x) for x in v], dtype=getattr(torch, t), device="cuda")


def tables(g, n_seq, ctx, page, spare=2):
    mp = -(-ctx // page)
    n_pages = n_seq * mp + spare
    return n_pages, g.permutation(n_pages)[:n_seq * mp].reshape(n_seq, mp).astype(np.int32)


def filled(shape, n_seq, ctx, page, seed=0, k_scale=None, v_scale=None):
    """A cache whose pages all hold codes as values get them and scales of
    about a thirtieth (times k_scale, v_scale of the block's number)."""
    heads, n_kv, qd, vd = shape
    g = np.random.default_rng(seed)
    n_pages, table = tables(g, n_seq, ctx, page)
    c = ref.Cache8(n_pages, n_kv, qd, vd, page, table)
    c.codes[:] = np.clip(np.rint(g.standard_normal(c.codes.shape, dtype=np.float32) * 37), -127, 127).astype(np.int8).view(np.uint8)
    c.scales[:] = g.uniform(0.02, 0.04, c.scales.shape)
    for i, f in enumerate((k_scale, v_scale)):
        if f is not None:
            c.scales[:, i] *= f(g, c.scales[:, i].shape)
    return c


_filled = {}


def shared(shape, n_seq, ctx, page):
    """filled(), kept for the tests that leave it alone."""
    key = (shape, n_seq, ctx, page)
    if key not in _filled:
        _filled.clear()
        _filled[key] = filled(*key)
    return _filled[key]


def on_gpu(c):
    import torch

    from moe_amd.paged import KvCache8

    n_seq = c.table.shape[0]
    b = KvCache8.sizes(c.n_pages, n_seq, n_kv=c.n_kv, qd=c.qd, vd=c.vd, page=c.page)
    assert b[:2] == (c.codes.size, c.scales.size * 4)
    return KvCache8(cuda(c.codes.reshape(-1)), cuda(c.scales.reshape(-1)), torch.zeros(b[2], dtype=torch.uint8, device="cuda"),
                    cuda(c.table), n_kv=c.n_kv, qd=c.qd, vd=c.vd, page=c.page)


def same_bytes(cache, c):
    codes = cache.codes.cpu().numpy().reshape(c.codes.shape)
    scales = cache.scales.cpu().numpy().reshape(c.scales.shape)
    assert np.array_equal(scales.view(np.uint32)[~np.isnan(c.scales)], c.scales.view(np.uint32)[~np.isnan(c.scales)])
    assert np.array_equal(np.isnan(scales), np.isnan(c.scales))
    assert np.array_equal(codes, c.codes), np.argwhere(codes != c.codes)[:5]


def rows_on_gpu(c, at, n_seq):
    """Rows of a step: each sequence's consecutive, in the order given."""
    from moe_amd.paged import Rows

    start, r = [], 0
    for s in range(n_seq + 1):
        while r < len(at) and at[r] is not None and at[r][0] < s:
            r += 1
        start.append(r)
    slot = [-1 if x is None else int(c.table[x[0], x[1] // c.page]) * c.page + x[1] % c.page for x in at]
    return Rows(ints(start), ints([-1 if x is None else x[0] for x in at]), ints([-1 if x is None else x[1] for x in at]),
                ints(slot, "int64"), ints([0] * n_seq))


def run_attend(cache, q, seq, pos, heads, scale, window=0, fill=7.0, max_pos=None, **kw):
    import torch

    out = torch.full((len(seq), heads * cache.vd), fill, device="cuda")
    cache.attend(cuda(q), ints(seq), ints(pos), out, max_pos=max(max(pos), 0) if max_pos is None else max_pos, scale=scale,
                 window=window, **kw)
    torch.cuda.synchronize()
    return out.cpu().numpy()


def close(got, want, tol=TOL):
    big = np.abs(want).max()
    err = np.abs(got - want).max() / (big if big > 0 else 1.0)
    assert err < tol, err


# ------------------------------------------------------------------ the write


def values(g, rows, width, kind):
    x = g.standard_normal((rows, width)).astype(np.float32) * np.exp(g.standard_normal((rows, 1))).astype(np.float32)
    if kind == "edges":  # zeros, halves of a step, values far below and above the rest, none at all
        x[::3] = np.rint(x[::3] * 4) / 4
        x[1::7] = 0
        x[2::11] *= np.float32(1e-34)
        x[3::13] *= np.float32(1e30)
        x.reshape(-1)[::97] = 0
    if kind == "bad":
        x.reshape(-1)[5::701] = np.inf
        x.reshape(-1)[9::907] = np.nan
    return x


@pytest.mark.parametrize("kind", ["plain", "edges", "bad"])
@pytest.mark.parametrize("page", [64, 256])
@pytest.mark.parametrize("shape", HEADS, ids=str)
def test_store_and_load(shape, page, kind):
    """Steps cut in every way: a block's codes and scale are those of its
    values, whatever wrote them; a step made again changes nothing; loads read
    what is held."""
    import torch

    heads, n_kv, qd, vd = shape
    g = np.random.default_rng(page + qd)
    n_seq, ctx = 3, 200
    n_pages, table = tables(g, n_seq, ctx, page)
    c = ref.Cache8(n_pages, n_kv, qd, vd, page, table)
    cache = on_gpu(c)
    length = [0, 0, 0]
    for step in ([70, 0, 5], [1, 16, 11], [1, 1, 1], [0, 15, 15], [30, 1, 17], [9, 32, 1], [1, 1, 1], [17, 63, 64]):
        at = [(s, length[s] + i) for s in range(n_seq) for i in range(step[s])] + [None]
        k, v = (values(g, len(at), n_kv * d, kind) for d in (qd, vd))
        c.store(at, k, v)
        rows = rows_on_gpu(c, at, n_seq)
        for _ in range(2):
            cache.store(cuda(k), cuda(v), rows)
            same_bytes(cache, c)
        length = [a + b for a, b in zip(length, step)]
    slots = [int(table[s, p // page]) * page + p % page for s in range(n_seq) for p in range(length[s])]
    want = [np.stack([np.concatenate([c.get(s, p, h, keys) for h in range(n_kv)]) for s in range(n_seq) for p in range(length[s])])
            for keys in (True, False)]
    k, v = torch.full((len(slots) + 2, n_kv * qd), 7.0, device="cuda"), torch.full((len(slots) + 2, n_kv * vd + 5), 7.0, device="cuda")
    cache.load(ints(slots + [-1, n_pages * page], "int64"), k, v[:, 2:2 + n_kv * vd])
    k, v = k.cpu().numpy(), v.cpu().numpy()
    # (a held value is the f32 product of code and scale: half a step of f32)
    np.testing.assert_allclose(k[:-2], want[0], rtol=2 ** -24, atol=2 ** -149)
    np.testing.assert_allclose(v[:-2, 2:2 + n_kv * vd], want[1], rtol=2 ** -24, atol=2 ** -149)
    assert (k[-2:] == 7).all() and (v[-2:] == 7).all() and (v[:, :2] == 7).all() and (v[:, 2 + n_kv * vd:] == 7).all()


def test_store_many_sequences():
    """Steps of few to many rows for each of 40 sequences are what the same rows
    give sequence by sequence."""
    import torch

    from moe_amd.paged import KvCache8

    n_kv, qd, vd, page, n_seq, ctx = 16, 64, 96, 64, 40, 330
    g = np.random.default_rng(5)
    n_pages, table = tables(g, n_seq, ctx, page)
    lay = ref.Cache8(1, n_kv, qd, vd, page, table)
    whole, parts = (KvCache8.new(n_pages, cuda(table), n_kv=n_kv, qd=qd, vd=vd, page=page) for _ in range(2))
    length = [0] * n_seq
    for most in (3, 7, 14, 33, 70, 1, 130):
        step = g.integers(0, most + 1, n_seq)
        at = [(s, length[s] + i) for s in range(n_seq) for i in range(step[s])]
        k, v = (cuda(values(g, len(at), n_kv * d, "mixed")) for d in (qd, vd))
        whole.store(k, v, rows_on_gpu(lay, at, n_seq))
        r = 0
        for s in range(n_seq):
            if step[s]:
                n = int(step[s])
                parts.store(k[r:r + n], v[r:r + n], rows_on_gpu(lay, at[r:r + n], n_seq))
                r += n
        assert torch.equal(whole.codes, parts.codes) and torch.equal(whole.scales, parts.scales), most
        length = [a + int(b) for a, b in zip(length, step)]


@pytest.mark.parametrize("shape", [(32, 8, 128, 128), (16, 16, 192, 128)], ids=str)
def test_load_many_rows_in_any_order(shape):
    """As rows read a few at a time: in order, turned round, shuffled, the same
    row twice, rows that are none between them."""
    import torch

    heads, n_kv, qd, vd = shape
    c = filled(shape, 5, 400, 128, seed=21)
    cache = on_gpu(c)
    g = np.random.default_rng(3)
    n = c.n_pages * c.page
    order = np.arange(1, 1025) % n
    for slots in (order, order[::-1], g.integers(0, n, 1024), np.where(g.random(1024) < 0.3, -1, order), np.repeat(order[:341], 3)[:1023]):
        many, few = ([torch.full((len(slots), n_kv * d), 7.0, device="cuda") for d in (qd, vd)] for _ in range(2))
        at = ints(slots, "int64")
        cache.load(at, *many)
        for r in range(0, len(slots), 50):
            cache.load(at[r:r + 50], *(x[r:r + 50] for x in few))
        for x, y in zip(many, few):
            assert torch.equal(x, y)


def test_store_large_steps():
    """More rows than one launch shape takes, in strides: as small steps."""
    import torch

    shape = (8, 2, 128, 64)
    heads, n_kv, qd, vd = shape
    g = np.random.default_rng(5)
    n_seq, ctx, page = 5, 2200, 64
    n_pages, table = tables(g, n_seq, ctx, page)
    c = ref.Cache8(n_pages, n_kv, qd, vd, page, table)
    cache, twin = on_gpu(c), on_gpu(c)
    length = [0] * n_seq
    for step in ([7, 0, 16, 1, 31], [2100, 900, 1, 0, 1333], [3, 3, 3, 3, 3]):
        at = [(s, length[s] + i) for s in range(n_seq) for i in range(step[s])]
        wide = torch.randn((len(at), n_kv * (qd + vd) + 3), device="cuda")
        k, v = wide[:, 1:1 + n_kv * qd], wide[:, 2 + n_kv * qd:2 + n_kv * (qd + vd)]
        cache.store(k, v, rows_on_gpu(c, at, n_seq))
        for r0 in range(0, max(step), 100):  # the twin: 100 rows of each sequence at a time
            some = [r for r, (s, p) in enumerate(at) if r0 <= p - length[s] < r0 + 100]
            twin.store(k[some], v[some], rows_on_gpu(c, [at[r] for r in some], n_seq))
        assert torch.equal(cache.codes, twin.codes) and torch.equal(cache.scales, twin.scales)
        length = [a + b for a, b in zip(length, step)]


def test_store_after_a_sequence_goes_back():
    """A sequence taken back into a block that is full: the earlier positions as
    they read; one that ends and begins again finds nothing of the old one."""
    import torch

    g = np.random.default_rng(3)
    c = ref.Cache8(4, 1, 64, 32, 64, np.array([[2, 0], [1, 3]], np.int32))
    cache = on_gpu(c)

    def step(s, p, n):
        at = [(s, p + i) for i in range(n)]
        k, v = values(g, n, 64, "plain"), values(g, n, 32, "plain")
        cache.store(cuda(k), cuda(v), rows_on_gpu(c, at, 2))
        return at, k, v

    c.store(*step(0, 0, 13))
    c.store(*step(0, 13, 30))     # block 0 fills
    c.store(*step(1, 0, 25))
    same_bytes(cache, c)
    for p in range(14):           # back into block 0, which is held no more: as it reads
        c.values[0, p] = tuple(np.stack([c.get(0, p, 0, keys)]).astype(np.float32) for keys in (True, False))
    c.store(*step(0, 14, 1))
    same_bytes(cache, c)
    c.store(*step(0, 15, 3))      # and on from there
    same_bytes(cache, c)
    c.store(*step(1, 0, 21))      # begun again, up to the block that was filling
    c.store(*step(1, 21, 2))
    c.store(*step(1, 20, 1))      # back in the block that is held: it knows 20 .. 22 of it
    same_bytes(cache, c)
    torch.cuda.synchronize()


# ------------------------------------------------------------------ attention


@pytest.mark.parametrize("name", ROWS)
@pytest.mark.parametrize("shape", HEADS, ids=str)
def test_attend(shape, name):
    heads, n_kv, qd, vd = shape
    c = shared(shape, 11, 300, 64)
    g = np.random.default_rng(1)
    seq, pos = [s for s, _ in ROWS[name]], [p for _, p in ROWS[name]]
    q = g.standard_normal((len(seq), heads * qd)).astype(np.float32)
    cache = on_gpu(c)
    for window in (0, 1, 20, 100):
        want = ref.attend(c, q, seq, pos, heads, qd ** -0.5, window, np.full((len(seq), heads * vd), 7.0))
        close(run_attend(cache, q, seq, pos, heads, qd ** -0.5, window), want)


@pytest.mark.parametrize("shape", [(8, 2, 64, 64), (32, 8, 128, 128), (16, 16, 192, 128), (6, 2, 96, 96), (40, 1, 64, 32)], ids=str)
@pytest.mark.parametrize("page,n,past", [(64, 1, 5000), (128, 3, 2900), (256, 200, 0), (64, 131, 1000), (64, 640, 0)])
def test_attend_long(shape, page, n, past):
    """Positions over several blocks, prompts over many, with a loose bound too."""
    heads, n_kv, qd, vd = shape
    c = filled(shape, 2, past + n + 70, page, seed=4)
    g = np.random.default_rng(2)
    rows = list(range(n)) if n < 20 else sorted(set(g.integers(0, n, 12).tolist() + [0, n - 1]))
    seq, pos = [1] * n + [0], list(range(past, past + n)) + [past // 2]
    q = g.standard_normal((len(seq), heads * qd)).astype(np.float32)
    cache = on_gpu(c)
    at = rows + [n]
    want = ref.attend(c, q[at], [seq[r] for r in at], [pos[r] for r in at], heads, qd ** -0.5)
    for bound in (past + n - 1, c.table.shape[1] * page - 1):
        close(run_attend(cache, q, seq, pos, heads, qd ** -0.5, max_pos=bound)[at], want)


def test_attend_many_sequences():
    """Decode steps of more sequences than blocks, a long prompt beside them."""
    shape = (32, 8, 128, 128)
    c = filled(shape, 40, 300, 64, seed=6)
    g = np.random.default_rng(3)
    rows = [(s, int(p)) for s, p in zip(range(39), g.integers(0, 300, 39))] + [(39, p) for p in range(290)]
    seq, pos = [s for s, _ in rows], [p for _, p in rows]
    q = g.standard_normal((len(seq), 32 * 128)).astype(np.float32)
    got = run_attend(on_gpu(c), q, seq, pos, 32, 128 ** -0.5)
    at = list(range(0, 39, 5)) + [39, 40, 102, 103, 200, 328]
    close(got[at], ref.attend(c, q[at], [seq[r] for r in at], [pos[r] for r in at], 32, 128 ** -0.5))


def powers(lo, hi):
    return lambda g, s: 2.0 ** g.integers(lo, hi + 1, s)


@pytest.mark.parametrize("k_scale,v_scale,scale", [
    (None, powers(-40, 0), 1.0), (None, powers(-12, 12), 1.0), (None, powers(-3, 90), 1.0), (None, powers(-80, -60), 1.0),
    (powers(-3, 1), powers(-20, 20), 1.0), (powers(-60, -58), None, 2.0 ** 60), (powers(60, 61), None, 2.0 ** -62),
    (powers(-2, 0), powers(0, 0), -1.0), (None, None, 0.0),
    (None, lambda g, s: g.integers(0, 2, s) * 1.0, 1.0), (lambda g, s: g.integers(0, 2, s) * 1.0, None, 1.0)], ids=range(11))
@pytest.mark.parametrize("name", ["decode", "chunk"])
def test_attend_uneven_scales(name, k_scale, v_scale, scale):
    """Blocks far larger and smaller than others, and of zeros.  Every output's
    own bar: 5e-6 of its weighted terms' size, sum of |weight x value|."""
    shape = heads, n_kv, qd, vd = (8, 2, 64, 64)
    c = filled(shape, 11, 300, 64, seed=7, k_scale=k_scale, v_scale=v_scale)
    g = np.random.default_rng(4)
    seq, pos = [s for s, _ in ROWS[name]], [p for _, p in ROWS[name]]
    q = g.standard_normal((len(seq), heads * qd)).astype(np.float32)
    s = np.float32(qd ** -0.5 * scale)
    want = ref.attend(c, q, seq, pos, heads, float(s))
    size = ref.Cache8(c.n_pages, n_kv, qd, vd, c.page, c.table)
    size.codes[:], size.scales[:] = c.codes, c.scales
    code = size.codes.view(np.int8)
    code[:, 64 * qd:] = np.abs(code[:, 64 * qd:])
    terms = ref.attend(size, q, seq, pos, heads, float(s))
    got = run_attend(on_gpu(c), q, seq, pos, heads, float(s))
    assert (np.abs(got - want) <= TOL * terms.max(1, keepdims=True) + 1e-37).all(), np.max(np.abs(got - want) / terms.max(1, keepdims=True))


def test_attend_sharp_scores():
    """Scores of up to about 100: a score's error is about 2^-23 of its terms'
    size, 40 here, so 5e-6 absolute at most and as much of the output."""
    shape = heads, n_kv, qd, vd = (32, 8, 128, 128)
    c = filled(shape, 3, 700, 64, seed=8)
    g = np.random.default_rng(5)
    seq, pos = [0, 1, 2] + [2] * 40, [699, 300, 0] + list(range(600, 640))
    q = g.standard_normal((len(seq), heads * qd)).astype(np.float32) * 20
    close(run_attend(on_gpu(c), q, seq, pos, heads, qd ** -0.5), ref.attend(c, q, seq, pos, heads, qd ** -0.5), 2e-5)


def test_attend_uneven_queries():
    """Heads of differing size in one row, of zeros, and with a few values far
    larger than the rest (each held to 2^-22 of the head's largest)."""
    shape = heads, n_kv, qd, vd = (8, 2, 64, 64)
    c = shared(shape, 11, 300, 64)
    g = np.random.default_rng(6)
    seq, pos = [0, 1, 2, 3], [299, 100, 17, 0]
    q = g.standard_normal((4, heads, qd)).astype(np.float32)
    q[:, 0] *= np.float32(1e-30)
    q[:, 1] = 0
    q[:, 2] *= np.float32(1e-3)
    q[:, 3, 5] *= 4
    q = q.reshape(4, -1)
    close(run_attend(on_gpu(c), q, seq, pos, heads, qd ** -0.5), ref.attend(c, q, seq, pos, heads, qd ** -0.5))


@pytest.mark.parametrize("name", ["decode", "chunk"])
def test_attend_not_a_number(name):
    """Blocks that read as NaN, behind a row's position or before its window,
    do not reach it; those it sees make it NaN.  Queries that are not finite
    make their own head NaN."""
    shape = heads, n_kv, qd, vd = (8, 2, 64, 64)
    c = filled(shape, 11, 300, 64, seed=9)
    seq, pos = [s for s, _ in ROWS[name]], [p for _, p in ROWS[name]]
    g = np.random.default_rng(7)
    q = g.standard_normal((len(seq), heads * qd)).astype(np.float32)
    for what in (0, 1):
        d = ref.Cache8(c.n_pages, n_kv, qd, vd, c.page, c.table)
        d.codes[:], d.scales[:] = c.codes, c.scales
        for s in range(11):  # blocks 2 and 9 (positions 32 and 144 on) of kv head 1
            for b in (2, 9):
                t = d.tile(s, 16 * b, 1)
                d.scales[t, what, b % 4] = np.nan
        cache = on_gpu(d)
        for window in (0, 20):
            got = run_attend(cache, q, seq, pos, heads, qd ** -0.5, window).reshape(len(seq), heads, vd)
            want = ref.attend(c, q, seq, pos, heads, qd ** -0.5, window).reshape(got.shape)
            for r, p in enumerate(pos):
                lo = max(0, p + 1 - window) if window else 0
                sees = any(lo <= 16 * b + 15 and 16 * b <= p for b in (2, 9))
                assert np.isnan(got[r, 4:]).all() == sees and not np.isnan(got[r, :4]).any()
                close(got[r, :4], want[r, :4])
                if not sees:
                    close(got[r, 4:], want[r, 4:])
    for bad in (np.inf, -np.inf, np.nan):
        x = q.copy().reshape(len(seq), heads, qd)
        x[0, 3, 60] = x[-1, 6, 0] = bad
        got = run_attend(on_gpu(c), x.reshape(q.shape), seq, pos, heads, qd ** -0.5).reshape(len(seq), heads, vd)
        hit = np.zeros((len(seq), heads), bool)
        hit[0, 3] = hit[-1, 6] = True
        assert np.isnan(got[hit]).all() and not np.isnan(got[~hit]).any()


def test_attend_pages_that_are_none():
    """Positions of pages outside the pool are not there; rows of nothing are 0."""
    shape = heads, n_kv, qd, vd = (8, 2, 64, 64)
    c = filled(shape, 3, 300, 64, seed=10)
    c.table[0, :2] = -1
    c.table[1, 2] = c.n_pages
    c.table[2, :] = -1
    seq, pos = [0, 0, 1, 2] + [0] * 30 + [1] * 30, [299, 100, 299, 50] + list(range(110, 140)) + list(range(180, 210))
    q = np.random.default_rng(8).standard_normal((len(seq), heads * qd)).astype(np.float32)
    cache = on_gpu(c)
    for window in (0, 40):
        want = ref.attend(c, q, seq, pos, heads, qd ** -0.5, window)
        got = run_attend(cache, q, seq, pos, heads, qd ** -0.5, window)
        close(got, want)
        assert (got[3] == 0).all() and (got[1] == 0).all()


def test_attend_strides_and_streams():
    """Rows inside wider ones, on a stream that is not current: what lies beside
    stays, and the result is the same bit for bit."""
    import torch

    shape = heads, n_kv, qd, vd = (8, 2, 96, 96)
    c = filled(shape, 11, 300, 64, seed=11)
    cache = on_gpu(c)
    for name in ("mixed", "chunk"):
        seq, pos = [s for s, _ in ROWS[name]], [p for _, p in ROWS[name]]
        n = len(seq)
        q = np.random.default_rng(9).standard_normal((n, heads * qd)).astype(np.float32)
        want = run_attend(cache, q, seq, pos, heads, 0.1)
        wq = torch.full((n, heads * qd + 7), float("nan"), device="cuda")
        wq[:, 3:3 + heads * qd] = cuda(q)
        wo = torch.full((n, heads * vd + 9), 7.0, device="cuda")
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        a, b = ints(seq), ints(pos)
        torch.cuda.synchronize()
        cache.attend(wq[:, 3:3 + heads * qd], a, b, wo[:, 5:5 + heads * vd], max_pos=max(pos), scale=0.1, stream=s)
        s.synchronize()
        got = wo.cpu().numpy()
        assert np.array_equal(got[:, 5:5 + heads * vd], want) and (got[:, :5] == 7).all() and (got[:, 5 + heads * vd:] == 7).all()


def test_attend_is_the_same_every_time():
    shape = heads, n_kv, qd, vd = (32, 8, 128, 128)
    c = filled(shape, 2, 3000, 64, seed=12)
    cache = on_gpu(c)
    q = np.random.default_rng(10).standard_normal((202, heads * qd)).astype(np.float32)
    seq, pos = [0] + [1] * 201, [2999] + list(range(700, 901))
    want = run_attend(cache, q, seq, pos, heads, 0.1)
    for _ in range(3):
        assert np.array_equal(run_attend(cache, q, seq, pos, heads, 0.1), want)


def test_pool_past_4_gib():
    """Pages whose codes lie behind 2^32 bytes are written, read and attended to
    as others are."""
    import torch

    from moe_amd.paged import KvCache8

    shape = heads, n_kv, qd, vd = (32, 8, 128, 128)
    page = 64
    each = 64 * n_kv * (qd + vd)
    n_pages = 2 ** 32 // each + 40
    table = torch.tensor([[n_pages - 1, 3, n_pages - 7], [0, 1, 2]], dtype=torch.int32, device="cuda")
    far = KvCache8.new(n_pages, table, n_kv=n_kv, qd=qd, vd=vd, page=page)
    near = KvCache8.new(8, torch.tensor([[7, 3, 4], [0, 1, 2]], dtype=torch.int32, device="cuda"), n_kv=n_kv, qd=qd, vd=vd, page=page)
    k, v, q = (torch.randn((150, n * 128), device="cuda") for n in (n_kv, n_kv, heads))
    at = [(0, p) for p in range(150)]
    got = []
    for cache in (far, near):
        c = ref.Cache8(1, n_kv, qd, vd, page, cache.table.cpu().numpy())
        rows = rows_on_gpu(c, at, 2)
        cache.store(k, v, rows)
        a, b, out = torch.empty_like(k), torch.empty_like(v), torch.empty((150, heads * vd), device="cuda")
        cache.load(rows.slot, a, b)
        cache.attend(q, rows.seq, rows.pos, out, max_pos=149, scale=0.1)
        got.append([x.cpu().numpy() for x in (a, b, out)])
    for x, y in zip(*got):
        assert np.array_equal(x, y)


@pytest.mark.parametrize("rows", [1, 3, 500])
def test_last_positions_there_are(rows):
    """Positions up to the last that 32 bits number, behind a window: results
    are those of the same rows a whole number of tiles earlier."""
    import torch

    from moe_amd.paged import KvCache8

    heads, n_kv, qd, vd, page, near_pages, window = 64, 8, 128, 128, 64, 27, 200
    far_pages = 2 ** 31 // page - 1
    k, v = (torch.randn((near_pages * page, n_kv * 128), device="cuda") for _ in range(2))
    q = torch.randn((rows, heads * qd), device="cuda")
    got = []
    for pages in (near_pages, far_pages):
        table = torch.full((1, pages), -1, dtype=torch.int32, device="cuda")
        table[0, -near_pages:] = torch.arange(near_pages, dtype=torch.int32, device="cuda")
        cache = KvCache8.new(near_pages, table, n_kv=n_kv, qd=qd, vd=vd, page=page)
        first = (pages - near_pages) * page
        at = [(0, first + p) for p in range(near_pages * page)]
        lay = type("Lay", (), dict(table=np.arange(-(pages - near_pages), near_pages, dtype=np.int32)[None], page=page))
        step = rows_on_gpu(lay, at, 1)
        cache.store(k, v, step)
        out = torch.full((rows, heads * vd), 7.0, device="cuda")
        cache.attend(q, step.seq[-rows:].contiguous(), step.pos[-rows:].contiguous(), out, max_pos=pages * page - 1, scale=0.1,
                     window=window)
        got.append((cache.codes.cpu().numpy(), cache.scales.cpu().numpy(), out.cpu().numpy()))
    for x, y in zip(*got):
        assert np.array_equal(x, y)


def test_captured_steps():
    """A decode step of tables, write and attention captured into a graph, with
    room for more rows than there are: every replay as the eager step."""
    import torch

    from moe_amd.paged import KvCache8, PageTable, Rows

    heads, n_kv, qd, vd = 8, 2, 64, 64
    kw = dict(n_kv=n_kv, qd=qd, vd=vd, page=64)
    n_seq, room = 3, 5
    made = []
    for _ in range(2):
        t = PageTable.new(n_seq, 6, 30, 64, "cuda")
        made.append((t, KvCache8.new(30, t.table, **kw), Rows.new(n_seq, room, "cuda"), torch.zeros((room, heads * vd), device="cuda")))
    add = torch.ones(n_seq, dtype=torch.int32, device="cuda")
    k, v, q = (torch.zeros((room, n * 64), device="cuda") for n in (n_kv, n_kv, heads))

    def step(t, cache, rows, out):
        t.advance(add, rows)
        cache.store(k, v, rows)
        cache.attend(q, rows.seq, rows.pos, out, max_pos=383, scale=0.125)

    def fill(i):
        g = torch.Generator(device="cuda").manual_seed(i)
        for x in (k, v, q):
            x.copy_(torch.randn(x.shape, generator=g, device="cuda"))

    # prompts of uneven lengths first
    for t, cache, rows, out in made:
        many = Rows.new(n_seq, 60, "cuda")
        t.advance(torch.tensor([40, 0, 20], dtype=torch.int32, device="cuda"), many)
        g = torch.Generator(device="cuda").manual_seed(99)
        cache.store(*(torch.randn((60, n_kv * 64), generator=g, device="cuda") for _ in range(2)), many)
    graph, (eager, captured) = torch.cuda.CUDAGraph(), made
    fill(0)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        step(*captured)
    torch.cuda.synchronize()
    for i in range(40):
        fill(i)
        graph.replay()
        step(*eager)
        torch.cuda.synchronize()
        assert torch.equal(eager[3], captured[3]) and torch.equal(eager[1].scales, captured[1].scales)
        assert torch.equal(eager[1].codes, captured[1].codes)
    assert eager[0].length.tolist() == [80, 40, 60]
