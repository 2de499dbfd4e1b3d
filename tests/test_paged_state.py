"""PagedState on the CPU: which rows a step has and which steps are refused,
with the device's tables replaced by a record of the calls."""
from types import SimpleNamespace

import pytest
import torch

from moe_amd import model as M
from moe_amd.model import Model, PagedState, Sparse, Spec


def fake_model(head_dim=64, layers=2, windows=()):
    m = Model.__new__(Model)
    m.spec = Spec(hidden=64, layers=layers, heads=4, kv_heads=2, head_dim=head_dim, vocab=10, windows=list(windows))
    m.device = torch.device("cpu")
    return m


@pytest.fixture
def state(monkeypatch):
    from moe_amd import _lib as L

    if not L.LIB_PATH.exists():
        from moe_amd.build import build

        build()
    st = fake_model().new_state(3, 100, cache="q4", page=32, pages=7)
    st.added = []
    monkeypatch.setattr(M.PageTable, "advance",
                        lambda self, add, rows, out=None, stream=None: (st.added.append((add.tolist(), len(rows.seq))), rows)[1])
    return st


def test_new_state_refuses():
    m = fake_model()
    for kw in (dict(cache="q8"), dict(pages=3), dict(sparse=Sparse(4)), dict(cache="q4", page=48), dict(cache="q4", pages=0),
               dict(cache="q4", sparse=Sparse(2, sinks=1, recent=2)), dict(cache="q4", sparse=Sparse(4, recent=0))):
        with pytest.raises(ValueError):
            m.new_state(2, 100, **kw)
    with pytest.raises(ValueError):
        fake_model(head_dim=40).new_state(2, 100, cache="q4")
    with pytest.raises(ValueError):
        m.new_state(0, 100, cache="q4")


def test_batch_orders_rows_by_sequence(state):
    b = state.batch([2, 0], [[7, 8, 9], [5]], torch.device("cpu"), 0, False)
    assert state.added == [([1, 0, 3], 4)]
    assert b.ids.tolist() == [5, 7, 8, 9] and b.ends == [3, 0] and b.max_pos == 2 and b.t == 4
    assert not b.sparse


def test_batch_refuses(state):
    go = lambda seqs, toks: state.batch(seqs, toks, torch.device("cpu"), 0, False)  # noqa: E731
    for seqs, toks in (([1, 1], [[1], [2]]), ([3], [[1]]), ([-1], [[1]]), ([0, 1], [[], []])):
        with pytest.raises(ValueError):
            go(seqs, toks)
    state.pos = [64, 90, 0]  # two and three of seven pages
    assert state.free_pages() == 2
    go([0, 2], [[1], [1] * 32])
    with pytest.raises(ValueError, match="pages"):
        go([0, 2], [[1], [1] * 33])
    assert state.pos == [64, 90, 0]


def test_sparse_steps_are_decode_steps(state):
    state.sparse = Sparse(4)
    go = lambda toks: state.batch([0, 1], toks, torch.device("cpu"), 0, False).sparse  # noqa: E731
    assert go([[1], [2]]) and not go([[1], [2, 3]])


def test_end(state):
    state.pos = [64, 90, 3]
    state.end([1])
    assert state.added == [([0, -1, 0], 0)] and state.pos == [64, 0, 3]
    with pytest.raises(ValueError):
        state.end([3])


def test_steps_are_not_captured(state, monkeypatch):
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    with pytest.raises(RuntimeError, match="captured"):
        state.batch([0], [[1]], torch.device("cpu"), 0, True)


def test_positions_have_numbers():
    with pytest.raises(ValueError):
        fake_model().new_state(1, 2 ** 31 - 1, cache="q4", pages=4)


def test_streams_of_another_device(state):
    with pytest.raises(ValueError, match="stream of cuda:1"):
        state.table._on(SimpleNamespace(device_index=1, cuda_stream=5))


class Sizes:
    """The library's sizes, its launches recorded: every workspace with the
    bytes that the call declares it to have."""

    def __init__(self, lib):
        self.lib, self.calls = lib, []

    def __getattr__(self, name):
        if name.endswith("_size"):
            return getattr(self.lib, name)
        if name in ("moe_kv4_attention", "moe_kv4_select"):
            return lambda *a: self.calls.append((name, *((a[14], a[15], a[9]) if "att" in name else (a[12], a[13], 0)))) or 0
        return lambda *a: 0


class Told:
    """A projection that does nothing."""

    def __call__(self, x, y, *a, **kw):
        return y

    def workspace_size(self, t):
        return 256

    feed_forward = __call__


def steps_of(monkeypatch, windows, sparse=None, pos=20000, rows=1):
    """Workspaces of one step's calls over layers with these windows: (call,
    declared bytes, bytes there are from its address on, window)."""
    from moe_amd import _lib as L

    m = fake_model(layers=len(windows), windows=windows)
    m.spec = Spec(hidden=64, layers=len(windows), heads=32, kv_heads=8, head_dim=128, vocab=10, windows=list(windows))
    st = m.new_state(1, pos + 64, cache="q4", sparse=sparse)
    st.pos[0] = pos
    m.embed = SimpleNamespace(offset=0, dt=0, rows=10, cols=64)
    m.store = SimpleNamespace(region=SimpleNamespace(device_ptr=lambda: 0))
    m.lm_head, m._ws, m._mws, m._ws_t, m.attn_scale, m.inv_freq = Told(), None, None, 0, 1.0, torch.zeros(64)
    m.layers = [dict(ln1=torch.ones(64), ln2=torch.ones(64), moe=Told(), q=Told(), k=Told(), v=Told(), o=Told(),
                     bias=[None] * 3, q_norm=None, k_norm=None, window=w) for w in windows]
    m._ffn_workspace = lambda t: torch.empty(256)
    lib, made = Sizes(L.lib()), []
    empty = torch.empty

    def record(*a, **kw):
        t = empty(*a, **kw)
        made.append(t)
        return t

    with monkeypatch.context() as p:
        p.setattr(M.L, "lib", lambda: lib)
        p.setattr(M, "_stream_ptr", lambda s: 0 if s is None else s)
        p.setattr(M.PageTable, "advance", lambda self, add, r, out=None, stream=None: r)
        p.setattr(torch, "empty", record)
        M.Model.trunk(m, [[1] * rows], st, stream=7)
    there = lambda at: max((t.data_ptr() + t.numel() * t.element_size() - at for t in made  # noqa: E731
                            if t.data_ptr() <= at < t.data_ptr() + t.numel() * t.element_size()), default=0)
    return [(name, n, there(at) if at else 0, w) for name, at, n, w in lib.calls], m, st


@pytest.mark.parametrize("windows", [(4096, None), (None, 4096), (2048, None), (1500, 9000, None, 64), (64, 64)], ids=str)
@pytest.mark.parametrize("sparse", [None, Sparse(16), Sparse(200, recent=3)], ids=str)
@pytest.mark.parametrize("rows", [1, 3])
def test_layers_of_different_windows_have_the_scratch_they_declare(monkeypatch, windows, sparse, rows):
    """A layer's workspace depends on its window and on lists: what a call
    says it has is there, and is what the call needs."""
    import ctypes as C

    from moe_amd import _lib as L

    calls, m, st = steps_of(monkeypatch, windows, sparse, rows=rows)
    assert [w for name, _, _, w in calls if "att" in name] == [w or 0 for w in windows]
    chosen = 0
    for name, declared, there, window in calls:
        assert declared <= there, f"{name}: {declared} bytes declared, {there} there (window {window})"
        need = C.c_uint64()
        if name == "moe_kv4_select":
            chosen = sparse.pages
            L.check(L.lib().moe_kv4_select_workspace_size(st.kv[0]._c, rows, 20000 + rows - 1, C.byref(need)))
        else:
            L.check(L.lib().moe_kv4_attention_workspace_size(st.kv[0]._c, rows, 32, 20000 + rows - 1, window, chosen,
                                                             C.byref(need)))
            chosen = 0
        assert declared >= need.value
    assert any(d for _, d, _, _ in calls) == (windows != (64, 64))


def test_steps_free_no_lengths(monkeypatch):
    """A step's new lengths and free pages go to memory that the state keeps:
    what one stream has yet to read is not freed for another to write."""
    from moe_amd import _lib as L

    m = fake_model()
    st = m.new_state(2, 100, cache="q4", page=32)
    where = lambda: (st.table.length.data_ptr(), st.table.state.data_ptr(), st.table.table.data_ptr(),  # noqa: E731
                     st.table.ring.data_ptr())
    m.spec.layers, m.layers = 0, []
    m.embed = SimpleNamespace(offset=0, dt=0, rows=10, cols=64)
    m.store = SimpleNamespace(region=SimpleNamespace(device_ptr=lambda: 0))
    m._workspace = m._ffn_workspace = lambda t: torch.empty(256)
    reads, writes = [], []

    def advance(self, add, r, out=None, stream=None):
        reads.append(self.length.data_ptr())
        writes.append(out.length.data_ptr())
        return r

    lib = Sizes(L.lib())
    monkeypatch.setattr(M.L, "lib", lambda: lib)
    monkeypatch.setattr(M, "_stream_ptr", lambda s: 0 if s is None else s)
    monkeypatch.setattr(M.PageTable, "advance", advance)
    seen = []
    for i in range(6):
        seen.append(where())
        kept = st.table.length
        M.Model.trunk(m, [[1], [2]], st, stream=7)
        assert st.table.length is not kept and reads[-1] == seen[-1][0] and writes[-1] == where()[0]
        del kept
    assert seen[0] != seen[1] and seen[0] == seen[2] == seen[4] and seen[1] == seen[3] == seen[5]
    assert seen[0][2:] == seen[1][2:]
    # a step that fails half-way leaves the state's own
    st.batch([0], [[1]], m.device, 7, False)
    assert where() == seen[0]


def test_windows_past_32_bits_are_as_wide_as_positions_go(monkeypatch):
    calls, _, _ = steps_of(monkeypatch, (2 ** 32 + 16, 64))
    assert [w for _, _, _, w in calls] == [2 ** 31 - 1, 64]
