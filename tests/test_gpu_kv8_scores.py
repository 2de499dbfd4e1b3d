"""Attention over the 8-bit cache with scores far larger than any weight's
range: one position takes all, and the row is that position's values.

Tolerance.  The largest score lies so far above the others (checked: 200 at
least, and 2e-5 of the sum of its terms' sizes, of which a score errs by 2^-22)
that their weights are 0 in any precision.  What is left is the value itself: its
weight in whole numbers, 2^-23, its scale, 2^-24, and three roundings of f32;
TOL is 40 times that."""
import numpy as np
import pytest

from gpu_util import TOL
from test_gpu_kv8 import close, filled, on_gpu, run_attend

pytestmark = pytest.mark.gpu

# name: (heads, kv heads, key width, value width), past, rows
CASES = {"decode": ((8, 2, 64, 64), 290, 1), "chunk": ((8, 2, 96, 96), 100, 40), "parts": ((4, 1, 128, 128), 20000, 1),
         "prompt": ((32, 8, 128, 128), 0, 640), "latent": ((16, 16, 192, 128), 200, 9), "large": ((4, 2, 256, 256), 300, 3)}


@pytest.mark.parametrize("sign", [1, -1, 0])
@pytest.mark.parametrize("size", [1e5, 1e6, 1e7, 1e8, 1e10, 1e20])
@pytest.mark.parametrize("name", CASES)
def test_one_position_takes_all(name, size, sign):
    """Scores about `size`, above zero, below, or on both sides."""
    shape, past, n = CASES[name]
    heads, n_kv, qd, vd = shape
    g = np.random.default_rng(int(np.log10(size)) + 2 + sign)
    c = filled(shape, 1, past + n, 64, seed=past)
    q = g.standard_normal((n, heads * qd)).astype(np.float32)
    if sign:
        keys = c.codes.view(np.int8)[:, :64 * qd]
        np.maximum(np.abs(keys), 1, out=keys)
        q = np.abs(q) * np.float32(sign)
    # (codes of about 30, scales of about 0.03)
    scale = float(np.float32(size / (qd if sign else qd ** 0.5)))
    pos = list(range(past, past + n))
    keys, vals = (c.span(0, past + n, which)[0] for which in (True, False))
    at, want = [], []
    rows = sorted({0, n // 2, n - 1})
    for r in rows:
        for h in range(heads):
            terms = keys[:pos[r] + 1, h // (heads // n_kv)] * (q[r, h * qd:(h + 1) * qd].astype(np.float64) * scale)
            s = terms.sum(1)
            top = int(s.argmax())
            rest = np.delete(s, top)
            if not len(rest) or s[top] - rest.max() > max(200, 2e-5 * np.abs(terms).sum(1).max()):
                at.append(r * heads + h)
                want.append(vals[top, h // (heads // n_kv)])
    assert len(at) > len(rows) * heads // 2
    got = run_attend(on_gpu(c), q, [0] * n, pos, heads, scale).reshape(n * heads, vd)[at]
    assert np.isfinite(got).all()
    close(got, np.stack(want))
