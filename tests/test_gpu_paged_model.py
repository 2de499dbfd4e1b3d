"""Whole decoders over the paged 4-bit cache (Model.new_state(cache="q4")).

The f32 path with its cache rows rounded to the same 4-bit values is the
reference: one decoder layer, so that both paths round the same rows and no
rounding error moves a code.  What differs is then the attention kernels'
summation order and the roundings after it: MODEL_TOL, the bar of whole-model
logits in f32 (gpu_util.py)."""
import numpy as np
import pytest

from gpu_util import MODEL_TOL, rel_err

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    import torch

    assert torch.cuda.is_available(), "no GPU visible"
    from moe_amd.layer import Context

    return Context(0)


def build(ctx, name, **kw):
    from moe_amd import synth
    from moe_amd.model import Model, Spec, upload_store

    shape = synth.model_shape(name, **kw)
    cfg, ck = synth.build_host_model(shape, 0)
    spec = Spec.derive(cfg, {n: t.shape for n, t in ck.items()})
    return Model(ctx, spec, upload_store(ctx, ck)), shape


SMALL = {"tiny_mixtral": dict(layers=1, vocab=1000),
         "v2_lite": dict(layers=1, vocab=1000, dense_inter=1408)}


@pytest.fixture(scope="module", params=list(SMALL))
def model(ctx, request):
    m, shape = build(ctx, request.param, **SMALL[request.param])
    yield m, shape
    m.close()


class Rounding:
    """The library with every row that goes into an f32 cache rounded to 4
    bits and back (through the host's quantiser)."""

    def __init__(self, lib, model):
        self.lib, (self.n_kv, self.qd, self.vd) = lib, model.kv_heads()

    def __getattr__(self, name):
        return getattr(self.lib, name)

    def _round(self, cache, width, rows):
        import ctypes as C

        import torch

        from moe_amd import _lib as L

        torch.cuda.synchronize()
        dst = _view(rows[0], (rows[1],), "<i8").long()
        # the whole cache up to the last row: addresses are rows of `width`
        n = int(dst.max()) + 1
        c = _view(cache, (n, width), "<f4")
        x = np.ascontiguousarray(c[dst].cpu().numpy())
        raw = np.empty((len(x), width // 32 * 18), np.uint8)
        L.check(self.lib.moe_quantize_rows(L.DT_Q4_0, x.ctypes.data_as(C.c_void_p), len(x), width, raw.ctypes.data_as(C.c_void_p)))
        L.check(self.lib.moe_dequant_rows(L.DT_Q4_0, raw.ctypes.data_as(C.c_void_p), len(x), width, x.ctypes.data_as(C.c_void_p)))
        c[dst] = torch.from_numpy(x).cuda()
        torch.cuda.synchronize()

    def moe_scatter_rows(self, src, rows, n, ss, dst, ds, dst_rows, sp):
        rc = self.lib.moe_scatter_rows(src, rows, n, ss, dst, ds, dst_rows, sp)
        self._round(dst, n, (dst_rows, rows))
        return rc

    def moe_mla_kv_store(self, kv, c, cs, lora, rows, heads, nope, rope, vd, kc, vc, dst_rows, sp):
        rc = self.lib.moe_mla_kv_store(kv, c, cs, lora, rows, heads, nope, rope, vd, kc, vc, dst_rows, sp)
        self._round(kc, heads * (nope + rope), (dst_rows, rows))
        self._round(vc, heads * vd, (dst_rows, rows))
        return rc


def _view(ptr, shape, kind):
    import torch

    class _V:
        __cuda_array_interface__ = {"shape": shape, "typestr": kind, "data": (ptr, False), "version": 3}

    return torch.as_tensor(_V(), device="cuda")


def rounded(model, monkeypatch, run):
    from moe_amd import model as M

    lib = M.L.lib()
    with monkeypatch.context() as p:
        p.setattr(M.L, "lib", lambda: Rounding(lib, model))
        return run()


def ids(n, vocab, seed):
    return [int(v) for v in np.random.default_rng(seed).integers(0, vocab, n)]


def test_steps_match_the_f32_cache(model, monkeypatch):
    """Prompts of several lengths at once, a chunk behind one of them, then
    decode steps, sequences in no order and some left out: logits as with an
    f32 cache of the same values."""
    m, shape = model
    calls = [([ids(70, shape.vocab, 1), ids(1, shape.vocab, 2), ids(33, shape.vocab, 3)], [2, 0, 1]),
             ([ids(40, shape.vocab, 4)], [2])]
    calls += [([[i], [i + 1], [i + 2]], [0, 1, 2] if i % 2 else [1, 2, 0]) for i in range(10, 14)]
    calls += [([[5], [6]], [2, 0])]

    def run(st):
        return [m.forward(t, st, seqs=s).cpu().numpy() for t, s in calls]

    want = rounded(m, monkeypatch, lambda: run(m.new_state(3, 128)))
    for page in (32, 64):
        got = run(m.new_state(3, 128, cache="q4", page=page))
        for a, b in zip(got, want):
            assert rel_err(a, b) < MODEL_TOL


def test_sparse_steps(model, monkeypatch):
    """Steps that choose among more pages than there are read everything;
    fewer change the logits and still run; prompts are never sparse."""
    from moe_amd.model import Sparse

    m, shape = model
    prompt, steps = ids(300, shape.vocab, 7), [[[11]], [[12]], [[13]]]

    def run(**kw):
        st = m.new_state(1, 400, cache="q4", page=32, **kw)
        return [m.forward(t, st).cpu().numpy() for t in [[prompt]] + steps]

    dense = run()
    for a, b in zip(run(sparse=Sparse(20)), dense):
        assert np.array_equal(a, b)
    few = run(sparse=Sparse(4, sinks=1, recent=2))
    assert np.array_equal(few[0], dense[0])
    assert all(np.isfinite(x).all() for x in few) and not np.array_equal(few[1], dense[1])


def test_pages_come_and_go(model):
    """More sequences over time than the pool holds at once; a step that
    wants more pages than are free is refused and changes nothing."""
    m, shape = model
    st = m.new_state(4, 128, cache="q4", page=32, pages=6)
    a, b = ids(90, shape.vocab, 1), ids(64, shape.vocab, 2)
    first = m.forward([a, b], st, seqs=[1, 3]).cpu().numpy()
    assert st.free_pages() == 1 and st.pos == [0, 90, 0, 64]
    with pytest.raises(ValueError, match="pages"):
        m.forward([ids(40, shape.vocab, 3)], st, seqs=[0])
    with pytest.raises(ValueError, match="once"):
        m.forward([[1], [2]], st, seqs=[1, 1])
    assert st.pos == [0, 90, 0, 64]
    st.end([1])
    assert st.free_pages() == 4
    m.forward([ids(100, shape.vocab, 3)], st, seqs=[0])
    st.end([0, 3])
    assert st.pos == [0] * 4 and st.free_pages() == 6
    # pages that others held, in another order: the same rows give the same logits
    again = m.forward([a, b], st, seqs=[0, 2]).cpu().numpy()
    assert rel_err(again, first) < MODEL_TOL


def test_a_failed_step_changes_nothing(model, monkeypatch):
    m, shape = model
    st, other = (m.new_state(1, 128, cache="q4", page=32) for _ in range(2))
    toks = ids(40, shape.vocab, 5)
    for s in (st, other):
        m.forward([toks], s)
    with monkeypatch.context() as p:
        p.setattr(type(m), "_ffn", staticmethod(lambda lay: (_ for _ in ()).throw(RuntimeError("half-way"))))
        with pytest.raises(RuntimeError):
            m.trunk([ids(50, shape.vocab, 6)], st)
    a, b = (m.forward([[3]], s).cpu().numpy() for s in (st, other))
    assert st.pos == other.pos == [41] and np.array_equal(a, b)


def test_generate_over_the_paged_cache(ctx):
    """The tiny Mixtral generates for prompts of several lengths at once."""
    m, shape = build(ctx, "tiny_mixtral")
    prompts = [ids(n, shape.vocab, n) for n in (5, 40, 16)]
    st = m.new_state(3, 96, cache="q4", page=32)
    out = m.generate_greedy(prompts, 24, st=st)
    assert [len(o) for o in out] == [24] * 3 and st.pos == [5 + 23, 40 + 23, 16 + 23]
    again = m.generate_greedy(prompts, 24, st=m.new_state(3, 96, cache="q4", page=64))
    # Page sizes change where rows lie, not what they hold.
    assert [o[:4] for o in again] == [o[:4] for o in out]
    m.close()


def test_a_context_past_the_f32_limit(ctx):
    """20000 positions: more than a row's scores an f32 state holds."""
    m, shape = build(ctx, "tiny_mixtral", layers=1, vocab=1000)
    with pytest.raises(ValueError):
        m.new_state(1, 20000)
    st = m.new_state(1, 20000, cache="q4")
    toks = ids(17000, 1000, 9)
    for i in range(0, 17000, 4250):
        x = m.forward([toks[i:i + 4250]], st)
    x = m.forward([[1]], st)
    assert st.pos == [17001] and np.isfinite(x.cpu().numpy()).all()
    m.close()


def test_ends_and_steps_on_a_stream_that_is_not_current(ctx):
    """What such a call leaves to its stream is not given to the current
    stream's next tensors while the stream is still behind."""
    import torch

    m, shape = build(ctx, "tiny_mixtral", **SMALL["tiny_mixtral"])
    st = m.new_state(4, 128, cache="q4", page=32)
    m.forward([ids(40, shape.vocab, 1), ids(33, shape.vocab, 2)], st)
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        torch.cuda._sleep(100_000_000)
    st.end([0], stream=s)
    b = st.batch([1, 2], [[1, 2], [3]], m.device, s.cuda_stream, False)
    junk = [torch.full((n,), 5, dtype=torch.int32, device="cuda") for n in (4, 5, 2, 3) for _ in range(50)]
    torch.cuda.synchronize()
    assert all((j == 5).all().item() for j in junk)
    assert st.table.length.tolist() == [0, 33, 0, 0] and b.table.length.tolist() == [0, 35, 1, 0]
    assert b.seq.tolist() == [1, 1, 2] and b.pos.tolist() == [33, 34, 0]
    m.close()


class Taking(Rounding):
    """The library with every row that goes into an f32 cache taken from a
    paged state's caches instead, as they read back: both attend over the same
    values, in any layer."""

    def __init__(self, lib, model, st):
        super().__init__(lib, model)
        self.st, self.calls = st, 0

    def moe_scatter_rows(self, src, rows, n, ss, dst, ds, dst_rows, sp):
        import torch

        st = self.st
        at = _view(dst_rows, (rows,), "<i8").long()
        cache, keys = st.kv[self.calls // 2], self.calls % 2 == 0
        self.calls += 1
        seq, pos = at // st.ctx, at % st.ctx
        slots = st.table.table[seq, pos // st.page].long() * st.page + pos % st.page
        x = torch.empty((rows, n), device="cuda")
        cache.load(slots, *((x, None) if keys else (None, x)))
        _view(dst, (int(at.max()) + 1, n), "<f4")[at] = x
        torch.cuda.synchronize()
        return 0


@pytest.mark.parametrize("windows", [(2048, None, 100), (None, 2600, 1500)], ids=str)
def test_layers_of_different_windows(ctx, monkeypatch, windows):
    """Decode steps past 3000 positions over layers whose windows differ, so
    that their positions are shared among differing numbers of blocks: logits as
    with an f32 cache of the same values."""
    from moe_amd import model as M
    from moe_amd import synth
    from moe_amd.model import Model, Spec, upload_store

    cfg, ck = synth.build_host_model(synth.model_shape("tiny_mixtral", layers=3, vocab=1000), 0)
    spec = Spec.derive(cfg, {n: t.shape for n, t in ck.items()})
    spec.windows = list(windows)
    m = Model(ctx, spec, upload_store(ctx, ck))
    paged, plain = m.new_state(1, 3200, cache="q4", page=32), m.new_state(1, 3200)
    lib = M.L.lib()
    for toks in [ids(3010, 1000, 3), [5], [6], ids(4, 1000, 4), [7]]:
        got = m.forward([toks], paged).cpu().numpy()
        with monkeypatch.context() as p:
            taking = Taking(lib, m, paged)
            p.setattr(M.L, "lib", lambda: taking)
            want = m.forward([toks], plain).cpu().numpy()
        assert taking.calls == 2 * len(windows)
        assert rel_err(got, want) < MODEL_TOL
    m.close()


@pytest.mark.parametrize("cache", ["f32", "q4"])
@pytest.mark.parametrize("late", ["current", "own"])
def test_steps_and_another_stream_do_not_wait_for_each_other(model, cache, late):
    """Prompts, decode steps and greedy tokens with stream= while the current
    stream, or that one, is behind: as without a stream, and the current
    stream's tensors as they were."""
    import torch

    m, shape = model
    prompts = [ids(40, shape.vocab, 1), ids(33, shape.vocab, 2)]
    kw = dict(cache="q4", page=32) if cache == "q4" else {}
    a, b = (m.new_state(2, 128, **kw) for _ in range(2))
    want = [m.forward(t, a).cpu().numpy() for t in (prompts, [[3], [4]])]
    tokens = m.generate_greedy(prompts, 4, m.new_state(2, 128, **kw))
    c = m.new_state(2, 128, **kw)
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(s if late == "own" else torch.cuda.current_stream()):
        torch.cuda._sleep(100_000_000)
    got = [m.forward(t, b, stream=s) for t in (prompts, [[3], [4]])]
    junk = [torch.full((n,), 5, dtype=torch.int32, device="cuda") for n in (4, 64, 5000, 100000) for _ in range(20)]
    assert m.generate_greedy(prompts, 4, c, stream=s.cuda_stream) == tokens
    s.synchronize()
    with torch.cuda.stream(s):
        got = [x.cpu().numpy() for x in got]
    for x, y in zip(got, want):
        assert np.array_equal(x, y)
    torch.cuda.synchronize()
    assert all((j == 5).all().item() for j in junk)
