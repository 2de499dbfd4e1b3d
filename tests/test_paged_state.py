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
