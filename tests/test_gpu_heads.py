"""Biases, head norms and rotation in one pass (moe_head_rope_rows): bit for bit
what moe_add_bias, moe_rmsnorm and moe_rope give in turn, and close to the
formula in 64 bits.

Tolerance of the formula: a value passes the bias, the scale, the weight and
the rotation, each a rounding of half a step of f32, and a norm whose sum of n
squares errs by sqrt(n) half steps at most; sine and cosine of the f32 angle err
by 2 of their own steps.  16 x 2^-24 of the pair's size covers that for heads of
up to 256; a whole projection's sum of up to 4096 squares is in chains of 16,
the same."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

TOL = 16 * 2.0 ** -24

#        heads, kv, width, offset, dim, n_inv
SHAPES = [(8, 2, 64, 0, 64, 32), (32, 8, 128, 0, 128, 64), (16, 16, 192, 128, 64, 32), (6, 2, 96, 0, 96, 48), (4, 4, 256, 0, 256, 128),
          (4, 1, 80, 0, 40, 20), (3, 1, 34, 2, 30, 15), (5, 5, 1, 0, 0, 0), (2, 1, 300, 20, 200, 100), (8, 2, 128, 0, 128, 50),
          (7, 7, 32, 0, 32, 40), (32, 4, 128, 64, 64, 32), (16, 2, 256, 0, 64, 32), (12, 3, 112, 0, 112, 56)]


def make(shape, rows, norm, bias, seed=0):
    import torch

    heads, kv, width, offset, dim, n_inv = shape
    g = torch.Generator(device="cuda").manual_seed(seed)
    n = lambda *s: torch.randn(s, generator=g, device="cuda")  # noqa: E731
    d = dict(q=n(rows, heads * width), k=n(rows, kv * width) * 3, v=n(rows, kv * 8),
             pos=torch.randint(0, 100000, (rows,), generator=g, device="cuda", dtype=torch.int32),
             inv=(10000.0 ** (-torch.arange(n_inv, device="cuda", dtype=torch.float64) / max(n_inv, 1))).float())
    if rows > 1:
        d["pos"][1] = 0
    kw = {}
    if norm:
        kw.update(q_norm=1 + 0.3 * n(width if norm == "head" else heads * width), k_norm=1 + 0.3 * n(width if norm == "head" else kv * width))
    if bias:
        kw.update(q_bias=n(heads * width), k_bias=n(kv * width), v_bias=n(kv * 8))
    return d, kw


def in_turn(shape, d, kw):
    """With the entry points of one step each."""
    import torch

    from moe_amd import _lib as L

    heads, kv, width, offset, dim, n_inv = shape
    lib, rows = L.lib(), len(d["pos"])
    out = []
    for name, h in (("q", heads), ("k", kv)):
        x = d[name].clone()
        if f"{name}_bias" in kw:
            L.check(lib.moe_add_bias(x.data_ptr(), x.numel(), kw[f"{name}_bias"].data_ptr(), h * width, None))
        w = kw.get(f"{name}_norm")
        if w is not None:
            y = torch.empty_like(x)
            n = w.numel()
            L.check(lib.moe_rmsnorm(x.data_ptr(), n, w.data_ptr(), x.numel() // n, n, 1e-6, y.data_ptr(), n, None))
            x = y
        if dim:
            L.check(lib.moe_rope(x.data_ptr(), rows, h * width, h, width, offset, dim, d["pos"].data_ptr(), d["inv"].data_ptr(), n_inv,
                                 None))
        torch.cuda.synchronize()
        out.append(x)
    return out


def formula(shape, d, kw):
    heads, kv, width, offset, dim, n_inv = shape
    out = []
    pos = d["pos"].cpu().numpy()
    ang = (pos.astype(np.float32)[:, None] * d["inv"].cpu().numpy()).astype(np.float64)  # the angle is the f32 product
    for name, h in (("q", heads), ("k", kv)):
        x = d[name].cpu().numpy().astype(np.float64)
        if f"{name}_bias" in kw:
            x = x + kw[f"{name}_bias"].cpu().numpy()
        w = kw.get(f"{name}_norm")
        if w is not None:
            n = w.numel()
            y = x.reshape(len(pos), -1, n)
            x = (y / np.sqrt((y * y).mean(-1, keepdims=True) + 1e-6) * w.cpu().numpy()).reshape(x.shape)
        x = x.reshape(len(pos), h, width).copy()
        half, m = dim // 2, min(dim // 2, n_inv)
        a, b = x[..., offset:offset + m].copy(), x[..., offset + half:offset + half + m].copy()
        c, s = np.cos(ang[:, None, :m]), np.sin(ang[:, None, :m])
        x[..., offset:offset + m], x[..., offset + half:offset + half + m] = a * c - b * s, a * s + b * c
        out.append(x.reshape(len(pos), -1))
    return out


@pytest.mark.parametrize("norm", [None, "head", "all"])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_rows(shape, bias, norm):
    import torch

    from moe_amd.heads import HeadRope

    heads, kv, width, offset, dim, n_inv = shape
    for rows in (1, 3, 70):
        d, kw = make(shape, rows, norm, bias)
        op = HeadRope(heads, kv, width, d["inv"], offset=offset, dim=dim, **kw)
        want = in_turn(shape, d, kw)
        # into rows inside wider ones; then in place
        wide = torch.full((rows, (heads + kv) * width + 9), 7.0, device="cuda")
        vo = torch.full((rows, kv * 8), 7.0, device="cuda")
        qo, ko = wide[:, 2:2 + heads * width], wide[:, 5 + heads * width:5 + (heads + kv) * width]
        q0, k0, v0 = d["q"].clone(), d["k"].clone(), d["v"].clone()
        more = dict(v=d["v"], v_out=vo) if bias else {}
        op(d["q"], d["k"], d["pos"], q_out=qo, k_out=ko, **more)
        assert torch.equal(qo, want[0]) and torch.equal(ko, want[1])
        assert torch.equal(d["q"], q0) and torch.equal(d["k"], k0)
        wide[:, 2:2 + heads * width] = wide[:, 5 + heads * width:5 + (heads + kv) * width] = 7.0
        assert (wide == 7).all()
        op(d["q"], d["k"], d["pos"], **(dict(v=d["v"]) if bias else {}))
        assert torch.equal(d["q"], want[0]) and torch.equal(d["k"], want[1])
        if bias:
            assert torch.equal(vo, v0 + kw["v_bias"]) and torch.equal(d["v"], vo)
        d["q"], d["k"], d["v"] = q0, k0, v0
        for got, exact in zip(want, formula(shape, d, kw)):
            got = got.cpu().numpy()
            x = exact.reshape(rows, -1, width)
            size = np.abs(x).copy()
            half, m = dim // 2, min(dim // 2, n_inv)
            pair = np.hypot(x[..., offset:offset + m], x[..., offset + half:offset + half + m])
            size[..., offset:offset + m] = size[..., offset + half:offset + half + m] = pair
            if bias:
                size = size + np.abs(size).max()  # (a sum that cancels)
            assert (np.abs(got.reshape(x.shape) - x) <= TOL * size + 1e-30).all()


def test_many_rows_and_streams():
    """Rows past one launch shape, rows of no position beside them, on another
    stream, captured."""
    import torch

    from moe_amd.heads import HeadRope

    shape = heads, kv, width, offset, dim, n_inv = (32, 8, 128, 0, 128, 64)
    d, kw = make(shape, 5003, "head", False)
    d["pos"][7] = -1
    op = HeadRope(heads, kv, width, d["inv"], **kw)
    want = in_turn(shape, d, kw)
    qo, ko = torch.empty_like(d["q"]), torch.empty_like(d["k"])
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    op(d["q"], d["k"], d["pos"], q_out=qo, k_out=ko, stream=s)
    s.synchronize()
    assert torch.equal(qo, want[0]) and torch.equal(ko, want[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        op(d["q"], d["k"], d["pos"], q_out=qo, k_out=ko)
    for i in range(4):
        d["q"].normal_()
        d["pos"].fill_(17 * i)
        graph.replay()
        torch.cuda.synchronize()
        want = in_turn(shape, d, kw)
        assert torch.equal(qo, want[0]) and torch.equal(ko, want[1])


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_not_a_number_stays_in_its_head(bad):
    import torch

    from moe_amd.heads import HeadRope

    shape = heads, kv, width, offset, dim, n_inv = (8, 2, 64, 0, 64, 32)
    d, kw = make(shape, 20, "head", True)
    d["q"][3, 64 * 5 + 7] = bad
    HeadRope(heads, kv, width, d["inv"], **kw)(d["q"], d["k"], d["pos"])
    got = d["q"].view(20, 8, 64)
    hit = torch.zeros((20, 8), dtype=torch.bool, device="cuda")
    hit[3, 5] = True
    assert got[3, 5].isnan().any() and not got[~hit].isnan().any() and not d["k"].isnan().any()
