"""Attention over the 8-bit cache where small values lie beside large ones: blocks
whose value scale is far below their neighbours', in dims of which the neighbours
have zeros.

Every output's own bar, of its own terms' size, sum of |weight x value|.  A weight
in whole numbers errs by half of 2^-23 of the largest product of weight and scale
among blocks whose scales lie within 2^5 of each other.  Scores here are within
log 4 (checked), so that is 2^-24 x 2^5 x 4 of the weights of the block with the
smallest scale, 7.6e-6, whatever the values; the scores' own errors and the roundings
of f32 add 2e-6."""
import numpy as np
import pytest

import kv8_reference as ref
from test_gpu_kv8 import filled, on_gpu, run_attend

pytestmark = pytest.mark.gpu

BAR = 1e-5
# (heads, kv heads, key width, value width), sequences' (first position, rows)
CASES = {"decode": ((8, 2, 64, 64), [(299, 1), (63, 1), (130, 1), (40, 1)]), "long": ((8, 1, 128, 128), [(5000, 1)]),
         "odd": ((6, 2, 96, 96), [(0, 40), (211, 1)]), "wide": ((4, 2, 256, 256), [(290, 2)]), "latent": ((16, 16, 192, 128), [(100, 9)]),
         "prompt": ((32, 8, 128, 128), [(0, 570)]), "prompt 64": ((48, 16, 64, 64), [(0, 1210)]),
         "prompt 192": ((64, 32, 192, 128), [(0, 650)])}


@pytest.mark.parametrize("far", [3, 6, 8, 12, 16, 20, 30, 60])
@pytest.mark.parametrize("name", CASES)
def test_dims_of_their_own(name, far):
    """Every block has one of four scales, 2^-far apart, and values in a quarter of
    the dims that is its scale's."""
    shape, runs = CASES[name]
    heads, n_kv, qd, vd = shape
    seq = [s for s, (p, n) in enumerate(runs) for _ in range(n)]
    pos = [p + i for p, n in runs for i in range(n)]
    c = filled(shape, len(runs), max(pos) + 1, 64, seed=far)
    g = np.random.default_rng(far)
    kind = g.integers(0, 4, c.scales.shape[::2])  # [tiles, blocks]
    kind[:, 1] = (kind[:, 0] + 1) % 4
    c.scales[:, 1] *= (2.0 ** -(np.minimum(far * kind, 90.0))).astype(np.float32)
    code = c.codes.view(np.int8)
    dim = np.arange(vd)
    for p in range(64):
        at = c._bytes(p, False)
        code[:, at] *= (dim[None] * 4 // vd == kind[:, p // 16, None]).astype(np.int8)
    q = g.standard_normal((len(seq), heads * qd)).astype(np.float32) * np.float32(0.1)
    scale = float(np.float32(qd ** -0.5))
    got = run_attend(on_gpu(c), q, seq, pos, heads, scale)
    rows = sorted({0, 1 % len(seq), len(seq) // 2, len(seq) - 1, max(0, len(seq) - 20)})
    args = (q[rows], [seq[r] for r in rows], [pos[r] for r in rows], heads, scale)
    for r in (rows[0], rows[-1]):
        k = c.span(seq[r], pos[r] + 1, True)[0]
        for h in range(heads):
            x = k[:, h // (heads // n_kv)] @ q[r, h * qd:(h + 1) * qd].astype(np.float64) * scale
            assert np.ptp(x) < np.log(4)
    want = ref.attend(c, *args)
    code[:, 64 * qd:] = np.abs(code[:, 64 * qd:])
    terms = ref.attend(c, *args)
    err = np.abs(got[rows] - want)
    assert (err <= BAR * terms + 1e-37).all(), np.max(err / np.maximum(terms, 1e-37))
