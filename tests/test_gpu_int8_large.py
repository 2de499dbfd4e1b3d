"""Products in 8-bit integers large enough for the kernels that go over blocks of
both operands in LDS: 64 x 128, 128 x 128 and 256 x 256 tokens by channels, over
every number of steps of 64 values about their rings' lengths, and past several
laps.  Bars as in test_gpu_int8.py; the whole-number sums are made in float64, which
holds them exactly."""
import numpy as np
import pytest

import kv8_reference as ref
from test_gpu_int8 import TOL, cuda, operands

pytestmark = pytest.mark.gpu

#         rows, channels (off every tile): what makes the rule in launch_product take each kernel
SIZES = {"64x128": (517, 2605), "128x128": (2043, 2101), "256x256": (3597, 3803)}


def exact(x, w):
    """In 64 bits, on the GPU."""
    (cx, sx), (cw, sw) = ref.quantise(x), ref.quantise(w)
    sums = cuda(cx).double() @ cuda(np.ascontiguousarray(cw.T)).double()
    return sums * cuda(sx).double()[:, None] * cuda(sw).double()


def near(got, want, size):
    err = (got.double() - want).abs()
    assert bool((err <= size).all()), float((err / size).max())


@pytest.mark.parametrize("k", [64, 65, 190, 256, 300, 384, 447, 512, 1000, 4159])
@pytest.mark.parametrize("name", SIZES)
def test_every_lap(name, k):
    import torch

    from moe_amd.int8 import Int8Linear

    t, n = SIZES[name]
    x, w = operands(t, n, k)
    want = exact(x, w)
    op, xd = Int8Linear(cuda(w)), cuda(x)
    y = torch.full((t, n), 7.0, device="cuda")
    op(xd, y)
    near(y, want, TOL * want.abs() + 1e-44)
    # rows inside wider ones, a residual, twice the same
    wide, res = torch.full((t, n + 5), 7.0, device="cuda"), torch.randn((t, n + 3), device="cuda")
    before = res.clone()
    op(xd, wide[:, 1:1 + n], residual=res[:, 2:2 + n])
    assert torch.equal(wide[:, 1:1 + n], y) and bool((wide[:, 0] == 7).all() and (wide[:, 1 + n:] == 7).all())
    total = before[:, 2:2 + n].double() + want
    near(res[:, 2:2 + n], total, TOL * want.abs() + 2.0 ** -24 * total.abs() * 1.0001 + 1e-44)
    assert torch.equal(res[:, :2], before[:, :2]) and torch.equal(res[:, 2 + n:], before[:, 2 + n:])


@pytest.mark.parametrize("name", SIZES)
def test_largest_sums_and_not_a_number(name):
    """Rows and channels of one sign (sums up to 127 x 127 x 4096), rows and channels
    of zeros, and ones that are NaN, which stay theirs."""
    import torch

    from moe_amd.int8 import Int8Linear

    t, n = SIZES[name]
    x, w = operands(t, n, 4096, seed=3)
    x[::3], w[::2] = np.abs(x[::3]).max(-1, keepdims=True), -np.abs(w[::2]).max(-1, keepdims=True)
    x[5], w[17] = 0, 0
    want = exact(x, w)
    x[t - 1, 4095], x[70, 0], w[n - 1, 63], w[130, 64] = np.nan, np.inf, -np.inf, np.nan
    for at in (t - 1, 70):
        want[at] = float("nan")
    for at in (n - 1, 130):
        want[:, at] = float("nan")
    y = torch.empty((t, n), device="cuda")
    Int8Linear(cuda(w))(cuda(x), y)
    assert torch.equal(y.isnan(), want.isnan())
    ok = ~want.isnan()
    near(y[ok], want[ok], TOL * want[ok].abs() + 1e-44)


@pytest.mark.parametrize("t,n", [(257, 8200), (8200, 257), (4099, 4800), (40, 50000), (9000, 40)])
def test_uneven_shapes(t, n):
    """Long in one direction: tiles dealt to the XCDs in bands that are not full."""
    import torch

    from moe_amd.int8 import Int8Linear

    x, w = operands(t, n, 200, seed=1)
    want = exact(x, w)
    y = torch.full((t, n), 7.0, device="cuda")
    Int8Linear(cuda(w))(cuda(x), y)
    near(y, want, TOL * want.abs() + 1e-44)
