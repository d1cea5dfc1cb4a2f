"""Products from several host threads and in graphs: no call's tokens meet another's.

More than eight tokens are quantised by a kernel before the product's; whatever another thread puts on the stream between the two, and whatever
another graph's replay does meanwhile, the product multiplies its own.
"""
import threading

import pytest
import torch

from mpserve_b200 import mx4

pytestmark = pytest.mark.gpu


def _weight(rows, cols, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return mx4.quantize(torch.randn((rows, cols), generator=g, device="cuda") * 0.02)


def _x(tokens, cols, seed, dtype=torch.bfloat16):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn((tokens, cols), generator=g, device="cuda").to(dtype)


@pytest.mark.parametrize("tokens", [9, 33, 64, 200])
def test_threads_on_one_stream(tokens):
    w = _weight(700, 1024, 1)
    xs = [_x(tokens, 1024, 10 + i) for i in range(4)]
    want = [(mx4.linear(x, w), mx4.gated_linear(x, w, w)) for x in xs]
    torch.cuda.synchronize()
    wrong, errors, start = [], [], threading.Barrier(len(xs))

    def serve(i):
        try:
            start.wait()
            got = [(mx4.linear(xs[i], w), mx4.gated_linear(xs[i], w, w)) for _ in range(150)]
            wrong.append(sum(not (torch.equal(a, want[i][0]) and torch.equal(b, want[i][1])) for a, b in got))
        except Exception as e:      # told by the test's thread
            errors.append(e)

    threads = [threading.Thread(target=serve, args=(i,)) for i in range(len(xs))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors and wrong == [0] * len(xs)
    assert mx4.product_timed_out() is False


@pytest.mark.parametrize("tokens", [9, 64, 200])
def test_graphs_captured_on_one_stream_and_replayed_on_two(tokens):
    w = _weight(700, 1024, 2)
    xs = [_x(tokens, 1024, 20 + i) for i in range(2)]
    want = [mx4.linear(x, w) for x in xs]
    graphs, ys = [], []
    for x in xs:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):                 # torch's own capture stream, the same for both
            ys.append([mx4.linear(x, w) for _ in range(20)])
        graphs.append(graph)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(10):
        for graph, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
        eager = [mx4.linear(x, w) for x in reversed(xs)]
        torch.cuda.synchronize()
        for y, right in zip(ys, want):
            assert all(torch.equal(one, right) for one in y)
        assert torch.equal(eager[0], want[1]) and torch.equal(eager[1], want[0])


def test_a_block_in_a_graph():
    w, d = _weight(640, 256, 3), _weight(256, 640, 4)
    block = mx4.GatedMlp(w, w, d, pre_weight=torch.ones(256, device="cuda"), next_weight=torch.ones(256, device="cuda"))
    h = _x(20, 256, 30)
    block(h)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        joined, n = block(h)
    h.copy_(_x(20, 256, 31))
    graph.replay()
    torch.cuda.synchronize()
    want = block(h)
    assert torch.equal(joined, want[0]) and torch.equal(n, want[1])


def test_a_record_is_seen_from_every_stream_once():
    """A wait that ran out in a product (the record is set by hand here) is told whichever stream asks: a replayed graph's products ran on another."""
    w = _weight(64, 64, 5)
    mx4.linear(_x(3, 64, 40), w)
    assert mx4.product_timed_out() is False
    mx4._workspaces[torch.cuda.current_device()][0] = 1
    torch.cuda.synchronize()
    with torch.cuda.stream(torch.cuda.Stream()):
        assert mx4.product_timed_out() is True
    assert mx4.product_timed_out() is False
