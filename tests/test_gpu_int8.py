"""Products in 8-bit integers on the GPU (moe_int8_*) against whole-number sums.

Codes and scales are defined with every step rounded to f32 and the sum of the
products is exact, so an output is (f32)sum * (scale * scale): three roundings,
half a step of f32 each, 3 x 2^-24 of itself and no more."""
import numpy as np
import pytest

import kv8_reference as ref

pytestmark = pytest.mark.gpu

TOL = 3 * 2.0 ** -24 * 1.0001


def cuda(x):
    import torch

    return torch.from_numpy(np.ascontiguousarray(x)).cuda()


def close(got, want, tol=TOL):
    err = np.abs(got.astype(np.float64) - want)
    assert (err <= tol * np.abs(want) + 1e-44).all(), float(np.nanmax(err / np.maximum(np.abs(want), 1e-30)))


SIZES = [(1, 1, 1), (1, 16, 64), (2, 17, 65), (1, 4096, 512), (3, 100, 31), (15, 33, 200), (16, 256, 128), (17, 130, 1000),
         (31, 576, 2048), (33, 255, 96), (64, 257, 257), (100, 1000, 320), (129, 300, 4100), (257, 513, 130), (300, 64, 64),
         (513, 640, 512), (1100, 1029, 192), (5, 20, 131072)]


def operands(t, n, k, seed=0):
    g = np.random.default_rng(seed + t * 7 + n)
    x = g.standard_normal((t, k)).astype(np.float32) * np.exp(g.standard_normal((t, 1))).astype(np.float32)
    w = g.standard_normal((n, k)).astype(np.float32) * 0.05
    return x, w


@pytest.mark.parametrize("t,n,k", SIZES)
def test_product(t, n, k):
    import torch

    from moe_amd.int8 import Int8Linear

    x, w = operands(t, n, k)
    op = Int8Linear(cuda(w))
    y = torch.full((t, n), 7.0, device="cuda")
    op(cuda(x), y)
    want = ref.product(x, w)
    close(y.cpu().numpy(), want)
    # rows inside wider ones, at odd addresses, with a residual
    wx, wy = torch.full((t, k + 5), float("nan"), device="cuda"), torch.full((t, n + 3), 7.0, device="cuda")
    wr = torch.randn((t, n + 9), device="cuda")
    wx[:, 1:1 + k], before = cuda(x), wr.cpu().numpy()
    op(wx[:, 1:1 + k], wy[:, 2:2 + n], residual=wr[:, 5:5 + n])
    got, after = wy.cpu().numpy(), wr.cpu().numpy()
    assert np.array_equal(got[:, 2:2 + n], y.cpu().numpy()) and (got[:, :2] == 7).all() and (got[:, 2 + n:] == 7).all()
    # (the sum rounds once more, or the product and the sum once together)
    sum_ = before[:, 5:5 + n].astype(np.float64) + want
    assert (np.abs(after[:, 5:5 + n] - sum_) <= TOL * np.abs(want) + 2.0 ** -24 * np.abs(sum_) * 1.0001 + 1e-44).all()
    after[:, 5:5 + n] = before[:, 5:5 + n]
    assert np.array_equal(after, before)


def test_every_size_of_few_rows():
    """Each number of rows about the kernels' tiles."""
    import torch

    from moe_amd.int8 import Int8Linear

    x, w = operands(150, 200, 448)
    want, op, xd = ref.product(x, w), Int8Linear(cuda(w)), cuda(x)
    for t in range(1, 151):
        y = torch.full((t, 200), 7.0, device="cuda")
        op(xd[:t], y)
        close(y.cpu().numpy(), want[:t])


@pytest.mark.parametrize("t,n", [(1, 640), (2, 640), (4, 640), (3, 5000), (9, 640), (90, 640), (700, 640)])
@pytest.mark.parametrize("place", ["y", "residual", "both"])
def test_results_in_the_inputs_memory(t, n, place):
    """y = x W^T or x += x W^T over x itself, whichever kernel takes the rows:
    what the blocks read is x as it was.  (Wider rows of y lie over x's.)"""
    import torch

    from moe_amd.int8 import Int8Linear

    k = 640
    x, w = operands(t, n, k, seed=9)
    op = Int8Linear(cuda(w))
    for _ in range(3):
        wide = torch.zeros((t, n), device="cuda")
        xd = wide[:, :k]
        xd.copy_(cuda(x))
        apart, before = torch.empty((t, n), device="cuda"), wide.cpu().numpy().astype(np.float64)
        want = ref.product(x, w)
        if place == "y":
            op(xd, wide)
            close(wide.cpu().numpy(), want)
            continue
        if place == "residual":
            op(xd, apart, residual=wide)
            close(apart.cpu().numpy(), want)
        else:  # half of x's row apart from the other half
            both = torch.zeros((t, 2 * n), device="cuda")
            xd = both[:, n - k // 2:n + k // 2]
            xd.copy_(cuda(x))
            before = both[:, n:].cpu().numpy().astype(np.float64)
            op(xd, both[:, :n], residual=both[:, n:])
            close(both[:, :n].cpu().numpy(), want)
            wide = both[:, n:]
        total = before + want
        assert (np.abs(wide.cpu().numpy() - total) <= TOL * np.abs(want) + 2.0 ** -24 * np.abs(total) * 1.0001 + 1e-44).all()


def test_largest_sums():
    """Every product 127 x 127 or its negative, over the widest rows: the sums'
    largest sizes."""
    import torch

    from moe_amd.int8 import Int8Linear

    x = np.ones((40, 131072), np.float32)
    x[1] = -1
    w = np.ones((20, 131072), np.float32) * 3
    w[7] *= -1
    y = torch.empty((40, 20), device="cuda")
    Int8Linear(cuda(w))(cuda(x), y)
    close(y.cpu().numpy(), ref.product(x, w))


def test_rows_of_every_kind():
    """Zeros, rows below 2^-100, values on halves of a step, huge ones; rows and
    channels with an infinity or a NaN are NaN, and no others."""
    import torch

    from moe_amd.int8 import Int8Linear

    x, w = operands(60, 90, 300, seed=4)
    x[3], x[4] = 0, x[4] * np.float32(1e-35)
    x[5] *= np.float32(1e25)
    x[6] = np.rint(x[6] * 2) / 2
    x[7, :] = 0
    x[7, 299] = 5
    w[8], w[9] = 0, w[9] * np.float32(1e-33)
    want = ref.product(x, w)
    x[10, 17], x[11, 0], x[12, 299] = np.inf, -np.inf, np.nan
    w[13, 299], w[14, 3] = np.nan, np.inf
    want[10:13] = np.nan
    want[:, 13:15] = np.nan
    for t in (60, 13):
        y = torch.empty((t, 90), device="cuda")
        Int8Linear(cuda(w))(cuda(x[:t]), y)
        got = y.cpu().numpy()
        assert np.array_equal(np.isnan(got), np.isnan(want[:t]))
        ok = ~np.isnan(want[:t])
        close(got[ok], want[:t][ok])


@pytest.mark.parametrize("t", [1, 40, 200])
def test_several_matrices_are_one_product(t):
    """Weights of several types, one behind the other: their products' columns."""
    import torch

    from moe_amd.int8 import Int8Linear

    x, w = operands(t, 333, 256, seed=5)
    parts = [cuda(w[:100]), cuda(w[100:117]).half(), cuda(w[117:332]).bfloat16(), cuda(w[332:])]
    op, xd = Int8Linear(parts), cuda(x)
    y = torch.empty((t, 333), device="cuda")
    op(xd, y)
    at = 0
    for p in parts:
        one = torch.empty((t, p.shape[0]), device="cuda")
        Int8Linear(p)(xd, one)
        assert torch.equal(one, y[:, at:at + p.shape[0]])
        close(one.cpu().numpy(), ref.product(x, p.float().cpu().numpy()))
        at += p.shape[0]


@pytest.mark.parametrize("dt", ["F32", "Q8_0", "Q5_0", "Q4_0"])
def test_views_of_a_checkpoint(dt):
    """Rows in a checkpoint's formats, as moe_dequant_rows reads them."""
    import ctypes as C

    import torch

    from moe_amd import _lib as L
    from moe_amd.int8 import Int8Linear
    from moe_amd.layer import Context, View

    d = {v: k for k, v in L.DT_NAMES.items()}[dt]
    x, w = operands(20, 70, 192, seed=6)
    p = lambda a: a.ctypes.data_as(C.c_void_p)  # noqa: E731
    raw = np.zeros(70 * L.lib().moe_row_bytes(d, 192), np.uint8)
    L.check(L.lib().moe_quantize_rows(d, p(w), 70, 192, p(raw)))
    L.check(L.lib().moe_dequant_rows(d, p(raw), 70, 192, p(w)))
    ctx = Context(0)
    region = ctx.upload(np.concatenate([np.zeros(256, np.uint8), raw]))
    each = len(raw) // 70
    views = [View(d, 30, 192, region.id, 256), View(d, 40, 192, region.id, 256 + 30 * each)]
    y = torch.empty((20, 70), device="cuda")
    Int8Linear.of_views(ctx, views, "cuda:0")(cuda(x), y)
    close(y.cpu().numpy(), ref.product(x, w))


def test_streams_and_graphs():
    """On a stream that is not current, and captured: every replay as the eager
    product of the rows as they are then."""
    import torch

    from moe_amd.int8 import Int8Linear

    for t in (1, 7, 300):
        x, w = operands(t, 200, 640, seed=7)
        op, xd = Int8Linear(cuda(w)), cuda(x)
        y, z = torch.empty((t, 200), device="cuda"), torch.empty((t, 200), device="cuda")
        op(xd, y)
        s = torch.cuda.Stream()
        torch.cuda.synchronize()
        op(xd, z, stream=s)
        s.synchronize()
        assert torch.equal(y, z)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            op(xd, z)
        for i in range(5):
            xd.copy_(torch.randn_like(xd) * (i + 1))
            graph.replay()
            op(xd, y)
            torch.cuda.synchronize()
            assert torch.equal(y, z)
