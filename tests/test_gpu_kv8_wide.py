"""Attention over the 8-bit cache at sizes where blocks take 64 columns (row, query
head) of one run: prompts and chunks of the widths that have such blocks, steps of
several runs beside them, with windows, blocks that read as NaN, pages that are not
there and uneven scales, against the plain 64-bit form on some of the rows (the
first and last of groups, ends of runs).  Bars as in test_gpu_kv8.py."""
import numpy as np
import pytest

import kv8_reference as ref
from gpu_util import TOL
from test_gpu_kv8 import close, filled, on_gpu, powers, run_attend

pytestmark = pytest.mark.gpu

# (heads, kv heads, key width, value width), rows from which on blocks of 64 columns are taken
SHAPES = {(32, 8, 128, 128): 560, (160, 2, 128, 128): 112, (48, 2, 128, 128): 374, (7, 7, 128, 128): 2560,
          (48, 16, 64, 64): 1200, (64, 32, 192, 128): 640}


def layout(shape, name):
    """Sequences and positions of a step's rows, more than SHAPES says."""
    n = SHAPES[shape]
    g = np.random.default_rng(n)
    if name == "prompt":
        return [(1, p) for p in range(n + 13)]
    if name == "chunk":
        return [(2, 333 + p) for p in range(n + 70)]
    if name == "any order":
        return [(0, int(p)) for p in g.permutation(n + 100)[:n + 9]]
    # several: prompts of uneven lengths, sequences that decode, rows that are none, two chunks of one sequence
    at, s = [], 3
    while len(at) < n + 150:
        k = int(g.choice([1, 1, 1, 2, 5, 17, 64, 150, 300]))
        first = int(g.integers(0, 200))
        at += [(s, first + i) for i in range(k)]
        if g.random() < 0.2:
            at += [(s, -1), (-1, 3), (99, 5)][:int(g.integers(1, 4))]
        s = 3 + (s - 2) % 9
    return at


def some(at, shape, g):
    """Rows worth a look: ends of runs and of groups, a few others."""
    rows = {0, 1, len(at) - 1, len(at) // 2} | set(g.integers(0, len(at), 4).tolist())
    ends = [r for r in range(1, len(at)) if at[r][0] != at[r - 1][0]]
    for r in g.permutation(ends)[:4]:
        rows |= {int(r) - 1, int(r)}
    rep = shape[0] // shape[1]
    tt = 64 // min(rep, 64)
    rows |= {min(len(at) - 1, x) for x in (tt - 1, tt, 5 * tt - 1, 5 * tt)}
    return sorted(rows)


def check(c, at, shape, window=0, tol=TOL, seed=0, scale=None, max_pos=None):
    heads, n_kv, qd, vd = shape
    g = np.random.default_rng(seed)
    q = g.standard_normal((len(at), heads * qd)).astype(np.float32)
    scale = float(np.float32(qd ** -0.5 if scale is None else scale))
    seq, pos = [s for s, _ in at], [p for _, p in at]
    got = run_attend(on_gpu(c), q, seq, pos, heads, scale, window, max_pos=max_pos)
    rows = some(at, shape, g)
    want = ref.attend(c, q[rows], [seq[r] for r in rows], [pos[r] for r in rows], heads, scale, window,
                      np.full((len(rows), heads * vd), 7.0))
    return got, rows, want


def context(at):
    return max(p for _, p in at) + 1


@pytest.mark.parametrize("name", ["prompt", "chunk", "any order", "several"])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_windows(shape, name):
    at = layout(shape, name)
    c = filled(shape, 12, context(at), 128, seed=2)
    for window in (0, 1, 20, 100, 700):
        got, rows, want = check(c, at, shape, window)
        close(got[rows], want)


@pytest.mark.parametrize("name", ["prompt", "several"])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_not_a_number(shape, name):
    """Blocks that read as NaN make the rows NaN that see them, and no others."""
    heads, n_kv, qd, vd = shape
    at = layout(shape, name)
    c = filled(shape, 12, context(at), 64, seed=3)
    for what in (0, 1):
        d = ref.Cache8(c.n_pages, n_kv, qd, vd, c.page, c.table)
        d.codes[:], d.scales[:] = c.codes, c.scales
        for s in range(12):  # positions 32 on and 144 on of the last kv head
            for b in (2, 9):
                if 16 * b < context(at):
                    d.scales[d.tile(s, 16 * b, n_kv - 1), what, b % 4] = np.nan
        for window in (0, 20):
            got, rows, _ = check(d, at, shape, window)
            clean, _, want = check(c, at, shape, window)
            hit = np.zeros((len(at), heads), bool)
            for r, (s, p) in enumerate(at):
                lo = max(0, p + 1 - window) if window else 0
                if p >= 0 and 0 <= s < 12:
                    hit[r, heads - heads // n_kv:] = any(lo <= 16 * b + 15 and 16 * b <= p for b in (2, 9))
            got, clean = got.reshape(len(at), heads, vd), clean.reshape(len(at), heads, vd)
            assert np.isnan(got[hit]).all() and not np.isnan(got[~hit]).any()
            close(clean.reshape(len(at), -1)[rows], want)
            close(got[~hit], clean[~hit])


@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_pages_that_are_none(shape):
    """Positions of pages outside the pool are not there, in the middle of a run, at
    its start and at its end; a query that is not finite is its head's alone."""
    heads, n_kv, qd, vd = shape
    at = layout(shape, "chunk")
    c = filled(shape, 12, context(at), 64, seed=4)
    c.table[2, [0, 3]], c.table[2, [1, 7]] = -1, c.n_pages
    for window in (0, 100):
        got, rows, want = check(c, at, shape, window)
        close(got[rows], want)
    c.table[2, :] = -1
    got, _, _ = check(c, at, shape)
    assert (got == 0).all()


@pytest.mark.parametrize("k_scale,v_scale,scale", [(None, powers(-40, 0), 1.0), (None, powers(-12, 12), 1.0), (None, powers(-80, -60), 1.0),
                                                   (powers(-3, 1), powers(-20, 20), 1.0), (powers(60, 61), None, 2.0 ** -62),
                                                   (None, None, -1.0), (None, lambda g, s: g.integers(0, 2, s) * 1.0, 1.0)],
                         ids=range(7))
@pytest.mark.parametrize("shape", [(32, 8, 128, 128), (48, 16, 64, 64), (64, 32, 192, 128)], ids=str)
def test_uneven_scales(shape, k_scale, v_scale, scale):
    """Every row's own bar: of the largest sum of |weight x value| in it."""
    heads, n_kv, qd, vd = shape
    at = layout(shape, "prompt")
    c = filled(shape, 2, context(at), 64, seed=5, k_scale=k_scale, v_scale=v_scale)
    got, rows, want = check(c, at, shape, scale=qd ** -0.5 * scale)
    code = c.codes.view(np.int8)
    code[:, 64 * qd:] = np.abs(code[:, 64 * qd:])
    _, _, terms = check(c, at, shape, scale=qd ** -0.5 * scale)
    assert (np.abs(got[rows] - want) <= TOL * terms.max(1, keepdims=True) + 1e-37).all()


@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_loose_bounds_and_again(shape):
    """A bound on the positions that is far above them, and the same bits every
    time."""
    at = layout(shape, "prompt")
    c = filled(shape, 2, context(at) + 500, 64, seed=6)
    got, rows, want = check(c, at, shape, max_pos=c.table.shape[1] * 64 - 1)
    close(got[rows], want)
    for _ in range(2):
        assert np.array_equal(check(c, at, shape)[0], got)
