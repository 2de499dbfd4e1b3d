"""Rows of a step that are to be skipped, in KvCache8.store: in front of a
sequence's other rows, behind them and between them.  Codes and scales are
compared for equality, as in test_gpu_kv8.py."""
import numpy as np
import pytest

import kv8_reference as ref
from test_gpu_kv8 import cuda, ints, on_gpu, same_bytes, tables, values

pytestmark = pytest.mark.gpu

HOW = ["slot -1", "slot past the pool", "no sequence", "sequence past the last", "position -1"]


def masked(c, start, at, skip, how):
    """A step's rows (sequence, position), those of `skip` made unusable."""
    from moe_amd.paged import Rows

    slot = [int(c.table[s, p // c.page]) * c.page + p % c.page for s, p in at]
    seq, pos = [s for s, _ in at], [p for _, p in at]
    for r in np.flatnonzero(skip):
        if how == "slot -1":
            slot[r] = -1
        if how == "slot past the pool":
            slot[r] = c.n_pages * c.page
        if how == "no sequence":
            seq[r] = -1
        if how == "sequence past the last":
            seq[r] = len(start) - 1
        if how == "position -1":
            pos[r] = -1
    return Rows(ints(start), ints(seq), ints(pos), ints(slot, "int64"), ints([0] * (len(start) - 1)))


def run(g, c, cache, length, step, skip, how):
    """sequence i: step[i] rows from length[i] on, of which skip[i] says which are skipped."""
    at = [(s, length[s] + i) for s in range(len(step)) for i in range(step[s])]
    flat = np.concatenate([np.asarray(x, bool) for x in skip]) if at else np.zeros(0, bool)
    k, v = (values(g, len(at), c.n_kv * d, "plain") for d in (c.qd, c.vd))
    c.store([None if skipped else x for x, skipped in zip(at, flat)], k, v)
    rows = masked(c, np.concatenate([[0], np.cumsum(step)]), at, flat, how)
    for _ in range(2):
        cache.store(cuda(k), cuda(v), rows)
        same_bytes(cache, c)


def setup(seed, n_seq=3, shape=(4, 2, 64, 96), ctx=700, page=128):
    _, n_kv, qd, vd = shape
    g = np.random.default_rng(seed)
    n_pages, table = tables(g, n_seq, ctx, page)
    c = ref.Cache8(n_pages, n_kv, qd, vd, page, table)
    return g, c, on_gpu(c)


@pytest.mark.parametrize("how", HOW)
@pytest.mark.parametrize("past", [0, 5, 21])
def test_last_and_first_rows(past, how):
    """Rows behind a sequence's end (padding) and rows that are there already:
    the step is as if it had the others alone."""
    g, c, cache = setup(past)
    if past:
        run(g, c, cache, [0, 0, 0], [past, past, 0], [[0] * past, [0] * past, []], how)
    a, b = [0] * 9, [0] * 9
    a[8], b[0] = 1, 1
    # (the first sequence's last row skipped, the second's first, which an earlier step wrote)
    run(g, c, cache, [past, max(past - 1, 0), 0], [9, 9, 9], [a, b if past else [0] * 9, [1] * 9], how)
    long = np.zeros(200, bool)
    long[90:] = True
    back = np.zeros(150, bool)
    end = max(past - 1, 0) + 9
    back[:end] = True  # all that is there, sent again
    run(g, c, cache, [past + 8, 0, 0], [200, 150, 70], [long, back, [0] * 70], how)
    run(g, c, cache, [past + 98, 150, 70], [40, 1, 3], [[0] * 40, [0], [0, 0, 1]], how)


@pytest.mark.parametrize("seed", range(6))
def test_rows_between(seed):
    """Rows skipped anywhere behind a sequence's first: their positions hold
    zeros in blocks that other rows are written to, and blocks without any stay
    as they were."""
    g, c, cache = setup(seed)
    step = [150, 37, 200]
    run(g, c, cache, [0, 0, 0], step, [[0] * n for n in step], HOW[0])
    skip = [g.random(n) < (0.1, 0.5, 0.9)[seed % 3] for n in step]
    skip[2][60:130] = True
    for x in skip:
        x[0] = False
    run(g, c, cache, [150, 37, 200], step, skip, HOW[seed % len(HOW)])


def test_many_rows():
    """As many rows as let a block of threads look at many of them, long skipped
    beginnings, and sequences without a row left."""
    g, c, cache = setup(11, n_seq=5, ctx=1400)
    step = [700, 701, 60, 650, 333]
    run(g, c, cache, [0] * 5, step, [[0] * n for n in step], HOW[0])
    skip = [np.zeros(n, bool) for n in step]
    skip[0][:600] = True
    skip[1][650:] = True
    skip[2][:] = True
    skip[3][100:500] = True
    skip[4][1::2] = True
    for x in range(592, 600):  # (a block of which codes are left)
        c.values[0, x] = tuple(np.stack([c.get(0, x, h, keys) for h in range(c.n_kv)]).astype(np.float32) for keys in (True, False))
    run(g, c, cache, [0, 701, 60, 650, 333], step, skip, HOW[1])
    run(g, c, cache, [700, 1351, 60, 1300, 666], [5] * 5, [[0] * 5] * 5, HOW[1])
