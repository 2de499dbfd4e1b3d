"""A model's biases and head norms on the CPU: sizes that do not fit its heads are
refused when it is made.  (The one pass over a step's rows writes as many values of
a row as its bias has.)"""
import pytest
import torch

from moe_amd.model import Model, Spec


def layer(**kw):
    m = Model.__new__(Model)
    m.spec = Spec(hidden=64, layers=1, heads=4, kv_heads=2, head_dim=16, vocab=10)
    m.inv_freq = torch.ones(8)
    one = dict(q=None, k=None, v=None, q_norm=None, k_norm=None)
    one.update(kw)
    return m._heads(dict(bias=[one["q"], one["k"], one["v"]], q_norm=one["q_norm"], k_norm=one["k_norm"]))


def test_sizes_that_fit():
    h = layer(q=torch.ones(64), k=torch.ones(32), v=torch.ones(32), q_norm=torch.ones(16), k_norm=torch.ones(32))
    assert (h.c.v_width, h.c.q_span, h.c.k_span) == (32, 1, 2)
    assert layer().c.v_width == 0


@pytest.mark.parametrize("name,n", [("v", 33), ("v", 31), ("v", 64), ("v", 16), ("q", 32), ("q", 65), ("k", 64), ("q_norm", 32),
                                    ("k_norm", 64), ("k_norm", 8)])
def test_sizes_that_do_not(name, n):
    with pytest.raises(ValueError):
        layer(**{name: torch.ones(n)})
