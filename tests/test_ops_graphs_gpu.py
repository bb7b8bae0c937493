"""The operators' scratch (GPU tests): a graph owns that of the calls that it
captured, a stream keeps what its calls need. The maps here take the two kernels of the group normalisation
that pass pairs through scratch."""

from contextlib import closing

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

SILU = 4


@pytest.fixture
def ops():
    from iec.ops import Ops

    o = Ops()
    yield o
    torch.cuda.synchronize()
    o.close()


def maps(seed, count, pixels=30000, c=256):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return [((k + 1) * torch.randn(1, pixels, c, generator=g, device="cuda") + k).half() for k in range(count)]


def capture(ops, stream, x, out):
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        ops.group_norm(x, 32, act=SILU, out=out)
    return graph


def test_graphs_of_one_stream_replay_at_once(ops):
    """Two graphs captured on one stream, replayed on two others beside calls
    on the capture stream: equal scratch would mix their statistics."""
    xs = maps(1, 3)
    want = [ops.group_norm(x, 32, act=SILU) for x in xs]
    outs = [torch.zeros_like(x) for x in xs]
    streams = [torch.cuda.Stream() for _ in xs]
    graphs = [capture(ops, streams[2], x, out) for x, out in zip(xs[:2], outs[:2])]
    torch.cuda.synchronize()
    for _ in range(200):
        for k in range(2):
            with torch.cuda.stream(streams[k]):
                graphs[k].replay()
        with torch.cuda.stream(streams[2]):
            ops.group_norm(xs[2], 32, act=SILU, out=outs[2])
    torch.cuda.synchronize()
    for out, y in zip(outs, want):
        assert torch.equal(out, y)
    for _ in range(200):  # each pass compared: a later right one does not hide a wrong one
        for k in range(2):
            with torch.cuda.stream(streams[k]):
                outs[k].zero_()
                graphs[k].replay()
        torch.cuda.synchronize()
        assert all(torch.equal(outs[k], want[k]) for k in range(2))


def test_branches_of_one_capture_run_at_once(ops):
    """Calls on two streams of one capture."""
    xs = maps(2, 2)
    want = [ops.group_norm(x, 32, act=SILU) for x in xs]
    outs = [torch.zeros_like(x) for x in xs]
    main, side = torch.cuda.Stream(), torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=main):
        side.wait_stream(main)
        with torch.cuda.stream(side):
            ops.group_norm(xs[1], 32, act=SILU, out=outs[1])
        ops.group_norm(xs[0], 32, act=SILU, out=outs[0])
        main.wait_stream(side)
    for _ in range(100):
        for out in outs:
            out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(out, y) for out, y in zip(outs, want))


def test_the_first_call_of_a_size_can_be_captured():
    """A capture needs no earlier call on its stream or of its size."""
    from iec.ops import Ops

    x = maps(3, 1, 20011, 288)[0]
    out = torch.zeros_like(x)
    with closing(Ops()) as ops:
        graph = capture(ops, torch.cuda.Stream(), x, out)
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone()
        assert torch.equal(got, ops.group_norm(x, 32, act=SILU))
        torch.cuda.synchronize()


def test_scratch_goes_with_its_graph(ops):
    """A program that captures again and again does not grow. 128 maps of 4097
    groups keep 4 MB of pairs."""
    g = torch.Generator(device="cuda")
    g.manual_seed(4)
    x = torch.randn(128, 3, 4097 * 3, generator=g, device="cuda").half()  # one value at a time: the two kernels
    out, side = torch.empty_like(x), torch.cuda.Stream()
    want = ops.group_norm(x, 4097)
    used = []
    for _ in range(40):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            ops.group_norm(x, 4097, out=out)
        graph.replay()
        torch.cuda.synchronize()
        del graph
        used.append(torch.cuda.mem_get_info()[0])
    assert torch.equal(out, want)
    assert used[3] - used[-1] < 32 << 20, [u >> 20 for u in used]


def test_a_stream_keeps_no_more_than_its_calls_need(ops):
    """300 streams, each with a map whose pairs take less than 128 KB."""
    x = maps(8, 1, 5000, 130)[0]  # channels that are no whole vectors: the two kernels
    out = torch.empty_like(x)
    ops.group_norm(x, 5, out=out)
    torch.cuda.synchronize()
    runtime = pytest.importorskip("cuda.bindings.runtime")  # (torch's own streams are a pool of 32)
    made = [runtime.cudaStreamCreateWithFlags(1) for _ in range(300)]
    assert all(err == runtime.cudaError_t.cudaSuccess for err, _ in made)
    before = torch.cuda.mem_get_info()[0]
    for _, s in made:
        ops.group_norm(x, 5, out=out, stream=int(s))
    torch.cuda.synchronize()
    kept = before - torch.cuda.mem_get_info()[0]
    for _, s in made:
        runtime.cudaStreamDestroy(s)
    assert kept < 100 << 20


def test_a_graph_outlives_larger_and_smaller_captures(ops):
    xs = maps(5, 1) + maps(6, 1, 90001) + maps(7, 1, 12345)
    side = torch.cuda.Stream()
    outs = [torch.zeros_like(x) for x in xs]
    graphs = [capture(ops, side, x, out) for x, out in zip(xs, outs)]
    del graphs[1]  # its scratch may be freed: the others' stays
    torch.cuda.synchronize()
    capture(ops, side, xs[1], outs[1]).replay()
    for k, graph in ((0, graphs[0]), (2, graphs[1])):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[k], ops.group_norm(xs[k], 32, act=SILU))
