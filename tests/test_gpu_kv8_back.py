"""Sequences of the 8-bit cache that are taken back to an earlier position, over
and over, and steps behind that are made again or made otherwise: what a block
gets are the values that were stored last, or, where only its codes are left, the
values that those read as.  Codes and scales are compared for equality, as in
test_gpu_kv8.py."""
import numpy as np
import pytest

import kv8_reference as ref
from test_gpu_kv8 import cuda, on_gpu, rows_on_gpu, same_bytes, tables, values

pytestmark = pytest.mark.gpu


class Steps:
    """A cache on the GPU and its plain form, written by the same steps."""

    def __init__(self, shape=(4, 2, 64, 96), n_seq=1, ctx=400, page=64, seed=0):
        _, n_kv, qd, vd = shape
        self.g = np.random.default_rng(seed)
        n_pages, table = tables(self.g, n_seq, ctx, page)
        self.c, self.n_seq = ref.Cache8(n_pages, n_kv, qd, vd, page, table), n_seq
        self.cache = on_gpu(self.c)

    def step(self, s, p, n, times=1, keep=True, size=1.0):
        """Positions p .. p + n - 1 of sequence s, `times` times over.  With
        keep false the plain form does not make the step."""
        at = [(s, p + i) for i in range(n)]
        k, v = (values(self.g, n, self.c.n_kv * d, "plain") * np.float32(size) for d in (self.c.qd, self.c.vd))
        if keep:
            self.c.store(at, k, v)
        rows = rows_on_gpu(self.c, at, self.n_seq)
        for _ in range(times):
            self.cache.store(cuda(k), cuda(v), rows)
            if keep:
                same_bytes(self.cache, self.c)

    def only_codes(self, s, p):
        """Of position p's block the positions before p are what they read as."""
        for x in range(p & ~15, p):
            self.c.values[s, x] = tuple(np.stack([self.c.get(s, x, h, keys) for h in range(self.c.n_kv)]).astype(np.float32)
                                        for keys in (True, False))


@pytest.mark.parametrize("first", [10, 16, 20])
@pytest.mark.parametrize("n", [13, 20, 45, 200])
@pytest.mark.parametrize("p", [4, 8, 9, 12, 15])
def test_back_twice_into_one_block(first, n, p):
    """Back to position 3, on over the block's end, and back into that block once
    more: its positions from 3 on are the second step's, of which codes are left,
    and none of the first's."""
    x = Steps(seed=first + n + p)
    x.step(0, 0, first)
    if first >= 16:
        x.only_codes(0, 3)
    x.step(0, 3, n)
    x.only_codes(0, p)
    x.step(0, p, 1)
    x.step(0, p + 1, 30)


def test_back_to_what_is_held():
    """Up to where an earlier step began the values themselves are known, also
    where the step after it went over the block's end."""
    x = Steps(seed=1)
    x.step(0, 0, 11)
    x.step(0, 11, 20)
    x.step(0, 9, 3)     # (held from the first step)
    x.step(0, 12, 40)
    x.step(0, 2, 1)
    x.step(0, 3, 70)


@pytest.mark.parametrize("n", [11, 12, 30, 100])
def test_again_behind_codes(n):
    """A step whose block's earlier positions are left as codes, made again: the
    same bytes, though what the codes read as is not what was stored."""
    for seed in range(4):
        x = Steps(shape=(8, 8, 64, 64), seed=seed)
        x.step(0, 0, 40, size=3.0)
        x.only_codes(0, 5)
        x.step(0, 5, n, times=3)


@pytest.mark.parametrize("n", [11, 30, 100])
def test_otherwise_behind_codes(n):
    """The same after such a step with far larger values that came to nothing:
    the block's earlier positions have lost nothing to them."""
    x = Steps(shape=(8, 8, 64, 64), seed=3)
    x.step(0, 0, 40)
    x.only_codes(0, 5)
    x.step(0, 5, n, keep=False, size=1e4)
    x.step(0, 5, n, times=2)
    x.step(0, 5 + n, 20)


def test_any_order():
    """Steps of any length from any earlier position, two sequences in turn: a
    model of what is known (the values of the block that is filling and of the one
    that the last step began in, up to where it began) says what a block gets."""
    x = Steps(shape=(4, 1, 32, 32), n_seq=2, ctx=400, seed=7)
    length, known = [0, 0], [{}, {}]  # block -> its positions whose values are known
    for _ in range(120):
        s = int(x.g.integers(0, 2))
        p = int(x.g.integers(max(0, length[s] - 40), length[s] + 1)) if x.g.random() < 0.6 else length[s]
        n = int(x.g.choice([1, 1, 2, 5, 16, 17, 40, 90]))
        if p + n > 380:
            p, n = 0, int(x.g.integers(1, 30))
        was, had = p // 16, p % 16
        if had and known[s].get(was, 0) < had:
            x.only_codes(s, p)
        x.step(s, p, n, times=2)
        last, filled = (p + n - 1) // 16, (p + n - 1) % 16 + 1
        known[s] = {was: had} if had else {}
        if filled < 16:
            known[s][last] = filled
        length[s] = p + n
