"""A layer's first calls on streams it has not seen, and one that makes a
workspace grow, are ordered with their own stream: the host does not wait for the
null stream, and what a call reads of its new workspace is cleared."""
import pytest
from test_gpu_new_streams import TOL, np, rel_err

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("name", ["tiny_mixtral", "v2_lite"])
def test_calls_do_not_wait_for_the_null_stream(name):
    """With a long kernel on the null stream: they return before it is done, and
    give the results of another layer's quiet ones."""
    import torch

    from moe_amd import synth
    from moe_amd.layer import Context

    host = synth.build_host_layer(synth.SHAPES[name], 3)
    ctx = Context(0)
    quiet, gl = synth.make_layer(ctx, host), synth.make_layer(ctx, host)
    xs = [torch.from_numpy(synth.activations(11 + t, t, host.shape.hidden)).cuda() for t in (24, 3, 1, 40)]
    streams = [torch.cuda.Stream() for _ in range(3)]
    streams.append(streams[2])

    def run(layer, x, stream):
        with torch.cuda.stream(stream):
            out = torch.full_like(x, float("nan"))
            layer.feed_forward(x, out, stream=stream)
        return out

    want = [run(quiet, x, s) for x, s in zip(xs, streams)]
    torch.cuda.synchronize()
    # memory that the workspaces get holds ones
    used = torch.full((1 << 28,), -1, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    del used
    torch.cuda.empty_cache()
    a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    done = torch.cuda.Event()
    with torch.cuda.stream(torch.cuda.default_stream()):
        torch.cuda._sleep(1_000_000)
        a.record()
        torch.cuda._sleep(10_000_000)
        b.record()
        b.synchronize()
        torch.cuda._sleep(int(10_000_000 * 1000 / a.elapsed_time(b)))  # a second
        done.record()
    got = [run(gl, x, s) for x, s in zip(xs, streams)]
    assert not done.query()  # (the null stream's kernel still runs)
    torch.cuda.synchronize()
    for w, g in zip(want, got):
        w, g = w.cpu().numpy(), g.cpu().numpy()
        assert np.isfinite(g).all() and rel_err(g, w) <= TOL


def test_growth_does_not_wait_for_other_streams():
    """Token counts that rise on several streams, streams dropped and others begun,
    with a long kernel on the null stream: calls return, and memory that changed
    hands gives what fresh memory does."""
    import torch

    from moe_amd import synth
    from moe_amd.layer import Context

    host = synth.build_host_layer(synth.SHAPES["tiny_mixtral"], 3)
    ctx = Context(0)
    quiet, gl = synth.make_layer(ctx, host), synth.make_layer(ctx, host)
    xs = [torch.from_numpy(synth.activations(11 + t, t, host.shape.hidden)).cuda() for t in (1, 24, 40, 100, 3, 200)]
    streams = [torch.cuda.Stream() for _ in range(4)]
    outs = [[torch.full_like(x, float("nan")) for x in xs] for _ in streams]
    want = [torch.empty_like(x) for x in xs]
    for x, out in zip(xs, want):
        quiet.feed_forward(x, out)
    for x in xs[:3]:  # memory to change hands
        gl.feed_forward(x, torch.empty_like(x), stream=streams[0])
    torch.cuda.synchronize()
    a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    done = torch.cuda.Event()
    torch.cuda._sleep(1_000_000)
    a.record()
    torch.cuda._sleep(10_000_000)
    b.record()
    b.synchronize()
    torch.cuda._sleep(int(10_000_000 * 1000 / a.elapsed_time(b)))  # a second
    done.record()
    for s, some in zip(streams, outs):
        for x, out in zip(xs, some):
            gl.feed_forward(x, out, stream=s)
    assert not done.query()  # (the null stream's kernel still runs)
    torch.cuda.synchronize()
    for some in outs:
        for w, g in zip(want, some):
            assert rel_err(g.cpu().numpy(), w.cpu().numpy()) <= TOL
    for s, some in zip(streams, outs):
        gl.release_stream(s)
        for x, w, out in zip(xs, want, some):
            out.fill_(float("nan"))
            gl.feed_forward(x, out)
            assert rel_err(out.cpu().numpy(), w.cpu().numpy()) <= TOL


def test_a_reservation_is_ready_when_it_returns():
    """A reserved stream's workspace is cleared by then, whatever the null stream
    does later: the first call may be a captured one that another stream replays."""
    import torch

    from moe_amd import synth
    from moe_amd.layer import Context

    host = synth.build_host_layer(synth.SHAPES["tiny_mixtral"], 3)
    gl = synth.make_layer(Context(0), host)
    x = torch.from_numpy(synth.activations(5, 24, host.shape.hidden)).cuda()
    want = torch.empty_like(x)
    gl.feed_forward(x, want)
    torch.cuda.synchronize()
    s, out = torch.cuda.Stream(), torch.full_like(x, float("nan"))
    gl.reserve(24, stream=s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        gl.feed_forward(x, out, stream=s)
    for _ in range(3):
        out.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        assert rel_err(out.cpu().numpy(), want.cpu().numpy()) <= TOL
