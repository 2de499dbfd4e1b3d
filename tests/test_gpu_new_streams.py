"""A layer's first calls on streams it has not seen: their workspaces are new
memory, which holds whatever was there, and begin with cleared counters."""
import numpy as np
import pytest

from gpu_util import TOL, rel_err

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("name", ["tiny_mixtral", "v2_lite"])
def test_first_calls_on_new_streams(name):
    """While another stream keeps the card busy, on memory that held ones: each
    stream's first call gives what a quiet one gives."""
    import torch

    from moe_amd import synth
    from moe_amd.layer import Context

    host = synth.build_host_layer(synth.SHAPES[name], 3)
    gl = synth.make_layer(Context(0), host)
    xs = [torch.from_numpy(synth.activations(11 + t, t, host.shape.hidden)).cuda() for t in (1, 24, 1, 200, 1, 3)]

    def run(x, stream):
        with torch.cuda.stream(stream):
            out = torch.full_like(x, float("nan"))
            gl.feed_forward(x, out, stream=stream)
        return out

    quiet = torch.cuda.Stream()
    want = []
    for x in xs:
        torch.cuda.synchronize()
        want.append(run(x, quiet))
    torch.cuda.synchronize()
    used = torch.full((1 << 28,), -1, dtype=torch.int32, device="cuda")
    busy, a = torch.cuda.Stream(), torch.randn((8192, 8192), device="cuda", dtype=torch.bfloat16)
    b = torch.empty_like(a)
    torch.cuda.synchronize()
    del used
    torch.cuda.empty_cache()
    with torch.cuda.stream(busy):
        for _ in range(20):
            torch.mm(a, a, out=b)
    got = [run(x, torch.cuda.Stream()) for x in xs]
    torch.cuda.synchronize()
    for w, g in zip(want, got):
        w, g = w.cpu().numpy(), g.cpu().numpy()
        assert np.isfinite(g).all() and rel_err(g, w) <= TOL
