"""Whole decoders whose attention runs in 8 bits: Model.new_state(cache="int8"),
Model(projections="int8").

One decoder layer, against the f32 path with what its cache holds replaced by
what the 8-bit cache holds: what differs is then the attention kernels'
summation order and the roundings after it, MODEL_TOL (gpu_util.py).  The 8-bit
projections are compared with the product's formula on the same inputs."""
import numpy as np
import pytest

import kv8_reference as ref
from gpu_util import MODEL_TOL, rel_err
from test_gpu_paged_model import SMALL, _view, build, ctx, ids  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", params=list(SMALL))
def model(ctx, request):  # noqa: F811
    m, shape = build(ctx, request.param, **SMALL[request.param])
    yield m, shape
    m.close()


class Holding:
    """The library with the f32 cache's rows, as its attention reads them,
    replaced by what blocks of 16 positions in 8 bits hold."""

    def __init__(self, lib):
        self.lib, self.calls = lib, 0

    def __getattr__(self, name):
        return getattr(self.lib, name)

    def moe_attention(self, q, qs, rows, heads, n_kv, qd, vd, scale, kc, vc, ctx, seq, pos, max_pos, window, out, os, sp):  # noqa: F811
        import torch

        torch.cuda.synchronize()
        last = {}
        for s, p in zip(_view(seq, (rows,), "<i4").tolist(), _view(pos, (rows,), "<i4").tolist()):
            last[s] = max(last.get(s, 0), p + 1)
        kept = []
        for at, d in ((kc, qd), (vc, vd)):
            c = _view(at, (max(last) + 1, ctx, n_kv, d), "<f4")
            kept.append((c, c.clone()))
            for s, n in last.items():
                x = np.zeros((-(-n // 16) * 16, n_kv, d), np.float32)
                x[:n] = c[s, :n].cpu().numpy()
                x = x.reshape(-1, 16, n_kv, d).transpose(0, 2, 1, 3)
                code, scales = ref.quantise(x.reshape(*x.shape[:2], -1))
                held = (code.astype(np.float32) * scales[..., None]).reshape(x.shape).transpose(0, 2, 1, 3).reshape(-1, n_kv, d)
                c[s, :n] = torch.from_numpy(np.ascontiguousarray(held[:n])).cuda()
        rc = self.lib.moe_attention(q, qs, rows, heads, n_kv, qd, vd, scale, kc, vc, ctx, seq, pos, max_pos, window, out, os, sp)
        torch.cuda.synchronize()
        for c, x in kept:  # (later rows change a block's codes: what the cache keeps is the values)
            c.copy_(x)
        torch.cuda.synchronize()
        self.calls += 1
        return rc


def held(monkeypatch, run):
    from moe_amd import model as M

    lib = Holding(M.L.lib())
    with monkeypatch.context() as p:
        p.setattr(M.L, "lib", lambda: lib)
        got = run()
    assert lib.calls
    return got


@pytest.mark.parametrize("page", [64, 128])
def test_steps_match_the_f32_cache(model, monkeypatch, page):
    """Prompts of several lengths at once, a chunk behind one of them, decode
    steps, sequences in no order and some left out, one that ends and begins
    again: logits as with an f32 cache of the same values."""
    m, shape = model
    calls = [([ids(70, shape.vocab, 1), ids(1, shape.vocab, 2), ids(33, shape.vocab, 3)], [2, 0, 1]),
             ([ids(40, shape.vocab, 4)], [2])]
    calls += [([[i], [i + 1], [i + 2]], [0, 1, 2] if i % 2 else [1, 2, 0]) for i in range(10, 14)]
    calls += [([[5], [6]], [2, 0]), ([ids(18, shape.vocab, 8)], [1])]

    def run(st):
        got = [m.forward(t, st, seqs=s).cpu().numpy() for t, s in calls]
        return got

    want = held(monkeypatch, lambda: run(m.new_state(3, 128)))
    st = m.new_state(3, 128, cache="int8", page=page)
    for _ in range(2):
        for a, b in zip(run(st), want):
            assert rel_err(a, b) < MODEL_TOL
        st.end([0, 1, 2])
    assert st.free_pages() == st.pages


def test_a_step_that_fails_is_as_if_not_made(model):
    """A step refused half-way, behind cache writes: made again, it gives what
    it would have given."""
    m, shape = model
    prompt, more = ids(29, shape.vocab, 1), ids(21, shape.vocab, 2)
    a, b = (m.new_state(1, 128, cache="int8") for _ in range(2))
    for st in (a, b):
        m.forward([prompt], st)
    lay = m.layers[0]
    kept = lay["o"]

    def fails(*args, **kw):
        raise RuntimeError("no")

    lay["o"] = fails
    with pytest.raises(RuntimeError):
        m.forward([more], b)
    lay["o"] = kept
    for toks in (more, [5]):
        assert np.array_equal(m.forward([toks], a).cpu().numpy(), m.forward([toks], b).cpu().numpy())


@pytest.mark.parametrize("name", list(SMALL))
def test_projections(ctx, name, monkeypatch):  # noqa: F811
    """8-bit projections with each cache: every product is the formula's on its
    inputs, through prompts and decode steps.  (The logits have no bar against
    f32 projections': a normal row's 8-bit values err by 0.8% of its size, so a
    score of s by about 0.011 s, and what scores of size s do to a random-init
    layer's logits has no bound but exp's.)"""
    from moe_amd import int8, model as M

    plain, shape = build(ctx, name, **SMALL[name])
    eight = M.Model(ctx, plain.spec, plain.store, projections="int8")
    calls = [[ids(40, shape.vocab, 1), ids(7, shape.vocab, 2)], [[3], [4]]]
    made = []
    call = int8.Int8Linear.__call__

    def keep(self, x, y, residual=None, stream=None):
        before = None if residual is None else residual.clone()
        call(self, x, y, residual=residual, stream=stream)
        made.append((self, x.clone(), y.clone(), before, None if residual is None else residual.clone()))
        return y

    monkeypatch.setattr(int8.Int8Linear, "__call__", keep)
    for cache in ("f32", "q4", "int8"):
        a, b = (m.new_state(2, 64, **({} if cache == "f32" else dict(cache=cache, page=64))) for m in (plain, eight))
        for t in calls:
            made.clear()
            want, got = plain.forward(t, a).cpu().numpy(), eight.forward(t, b).cpu().numpy()
            assert len(made) == (2 if plain.spec.mla is None else 4 if plain.spec.mla.q_lora == 0 else 5)
            assert np.isfinite(got).all() and not np.array_equal(got, want)
            for op, x, y, before, after in made:
                code = op.packed[: -(-op.n // 16) * 16 * (-(-op.k // 64) * 64)].cpu().numpy().view(np.int8)
                code = code.reshape(-(-op.n // 16), -1, 4, 16, 16).transpose(0, 3, 1, 2, 4).reshape(-(-op.n // 16) * 16, -1)[: op.n, : op.k]
                sw = op.packed[-(-op.n // 16) * 16 * (-(-op.k // 64) * 64):].cpu().numpy().view(np.float32)[: op.n].astype(np.float64)
                cx, sx = ref.quantise(x.cpu().numpy())
                exact = (cx.astype(np.int64) @ code.astype(np.int64).T) * (sx.astype(np.float64)[:, None] * sw)
                assert (np.abs(y.cpu().numpy() - exact) <= 3.001 * 2.0 ** -24 * np.abs(exact)).all()
                if before is not None:
                    sum_ = before.double().cpu().numpy() + exact
                    assert (np.abs(after.cpu().numpy() - sum_) <= 3.001 * 2.0 ** -24 * np.abs(exact) + 1.001 * 2.0 ** -24 * np.abs(sum_)).all()
    eight.close()
    plain.close()


def test_refuses():
    from moe_amd import model as M

    with pytest.raises(ValueError):
        M.Model(None, None, None, projections="int4")


def test_steps_and_another_stream_do_not_wait_for_each_other(model):
    """Prompts, decode steps and greedy tokens with stream= while the current
    stream is behind: as without a stream."""
    import torch

    m, shape = model
    prompts = [ids(40, shape.vocab, 1), ids(33, shape.vocab, 2)]
    kw = dict(cache="int8", page=64)
    a, b, c = (m.new_state(2, 128, **kw) for _ in range(3))
    want = [m.forward(t, a).cpu().numpy() for t in (prompts, [[3], [4]])]
    tokens = m.generate_greedy(prompts, 4, m.new_state(2, 128, **kw))
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    torch.cuda._sleep(100_000_000)
    got = [m.forward(t, b, stream=s) for t in (prompts, [[3], [4]])]
    assert m.generate_greedy(prompts, 4, c, stream=s.cuda_stream) == tokens
    s.synchronize()
    with torch.cuda.stream(s):
        got = [x.cpu().numpy() for x in got]
    for x, y in zip(got, want):
        assert np.array_equal(x, y)
