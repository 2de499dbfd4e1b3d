"""8-bit products and models made under a stream that is behind: they are finished
when their constructor returns, so a first call may go to any other stream."""
import numpy as np
import pytest

import kv8_reference as ref
from test_gpu_int8 import close, cuda, operands
from test_gpu_paged_model import SMALL, build, ctx, ids  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("t", [2, 50])
def test_a_product_is_ready_when_it_is_made(t):
    import torch

    from moe_amd.int8 import Int8Linear

    x, w = operands(t, 600, 512)
    xd, wd, y = cuda(x), cuda(w), torch.full((t, 600), 7.0, device="cuda")
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(a):
        torch.cuda._sleep(100_000_000)
        op = Int8Linear(wd)
        done = torch.cuda.Event()
        done.record()
    op(xd, y, stream=b)
    b.synchronize()
    close(y.cpu().numpy(), ref.product(x, w))
    assert done.query()


@pytest.mark.parametrize("name", list(SMALL))
def test_a_model_is_ready_when_it_is_made(ctx, name):  # noqa: F811
    import torch

    from moe_amd import model as M

    plain, shape = build(ctx, name, **SMALL[name])
    prompt = [ids(20, shape.vocab, 1)]
    made = []
    for _ in range(2):
        m = M.Model(ctx, plain.spec, plain.store, projections="int8")
        made.append(m.forward(prompt, m.new_state(1, 64)).cpu().numpy())
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(b):
        st = m.new_state(1, 64)
    with torch.cuda.stream(a):
        torch.cuda._sleep(100_000_000)
        m = M.Model(ctx, plain.spec, plain.store, projections="int8")
    got = m.forward(prompt, st, stream=b)
    b.synchronize()
    assert np.array_equal(got.cpu().numpy(), made[0]) and np.array_equal(*made)
    plain.close()
