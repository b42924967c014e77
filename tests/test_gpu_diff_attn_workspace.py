"""Differential attention whose keys are split over the workspace: calls that run at the same time, in graphs, on streams that
share a handle and on threads, never share their sums."""
import threading

import pytest
import torch

import tsn

pytestmark = pytest.mark.gpu
PER_THREAD = 2   # cudaStreamPerThread: one handle, a stream for each thread


class Calls:
    """Calls of one token over many keys, each with queries, results and parts of its own, and what they give."""

    def __init__(self, n=4):
        g = torch.Generator(device="cuda")
        g.manual_seed(5)
        r = lambda *s: torch.randn(s, generator=g, device="cuda")  # noqa: E731
        self.lams, self.w = [0.1 * r(64) for _ in range(4)], 1 + 0.1 * r(128)
        self.k, self.v = (r(1, 30000, 8, 128).bfloat16() for _ in range(2))
        # other lengths, so that their parts are of other numbers and sizes
        self.keys = [30000 - 7000 * i for i in range(n)]
        self.q = [(1.2 * r(1, 1 + i, 8, 128)).bfloat16() for i in range(n)]
        self.out = [torch.empty_like(q) for q in self.q]
        dev = tsn.Device(0, stream=torch.cuda.current_stream().cuda_stream)
        op = self.op(dev)
        for i in range(n):
            self.call(op, i)
        dev.commit()
        torch.cuda.synchronize()
        self.want = [o.clone() for o in self.out]
        self.clear()
        dev.close()

    def op(self, dev):
        return tsn.DiffAttention(dev, 64, *self.lams, lambda_init=0.4, norm_weight=self.w)

    def call(self, op, i, out=None):
        n = self.keys[i]
        op(self.q[i], self.k[:, :n], self.v[:, :n], self.out[i] if out is None else out)

    def clear(self):
        for o in self.out:
            o.fill_(float("nan"))
        torch.cuda.synchronize()

    def right(self, *which):
        torch.cuda.synchronize()
        return all(torch.equal(self.out[i], self.want[i]) for i in which)


@pytest.fixture(scope="module")
def calls():
    return Calls()


def on(dev, stream):
    tsn.check(tsn.lib().tsn_device_set_stream(dev.h, stream.cuda_stream if isinstance(stream, torch.cuda.Stream) else stream))


def test_a_first_call_can_be_captured(calls):
    calls.clear()
    side = torch.cuda.Stream()
    dev = tsn.Device(0, stream=side.cuda_stream)
    op = calls.op(dev)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        calls.call(op, 0)
    for _ in range(3):
        calls.clear()
        g.replay()
        assert calls.right(0)
    del g
    torch.cuda.synchronize()
    dev.close()


def test_replays_beside_replays_and_calls(calls):
    streams = [torch.cuda.Stream() for _ in range(3)]
    dev = tsn.Device(0, stream=streams[0].cuda_stream)
    op, graphs = calls.op(dev), []
    for i, s in enumerate(streams[:2]):
        on(dev, s)
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1], stream=s):
            for _ in range(5):
                calls.call(op, i)
    on(dev, streams[2])
    for _ in range(10):
        calls.clear()
        for _ in range(4):
            for g, s in zip(graphs, streams):
                with torch.cuda.stream(s):
                    g.replay()
            calls.call(op, 2)
        assert calls.right(0, 1, 2)
    graphs.clear()
    torch.cuda.synchronize()
    dev.close()


def test_branches_of_a_capture(calls):
    """Calls on two streams that a capture forks and joins are nodes without an order between them."""
    main, fork = torch.cuda.Stream(), torch.cuda.Stream()
    dev = tsn.Device(0, stream=main.cuda_stream)
    op = calls.op(dev)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=main):
        fork.wait_stream(main)
        for _ in range(4):
            on(dev, main)
            calls.call(op, 0)
            on(dev, fork)
            calls.call(op, 3)
        main.wait_stream(fork)
    on(dev, main)
    for _ in range(10):
        calls.clear()
        g.replay()
        assert calls.right(0, 3)
    del g
    torch.cuda.synchronize()
    dev.close()


def test_threads_with_a_stream_each(calls):
    """One handle on the per-thread default stream: the same handle value is another stream in each thread."""
    dev = tsn.Device(0, stream=PER_THREAD)
    outs = [[torch.empty_like(calls.q[i]) for _ in range(50)] for i in range(3)]
    torch.cuda.synchronize()
    errors = []

    def run(i):
        try:
            op = calls.op(dev)
            for o in outs[i]:
                calls.call(op, i, o)
        except Exception as e:   # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=run, args=(i,)) for i in range(3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not errors
    assert all(torch.equal(o, calls.want[i]) for i in range(3) for o in outs[i])
    dev.close()


def test_graphs_give_their_workspaces_back(calls):
    side = torch.cuda.Stream()
    dev = tsn.Device(0, stream=side.cuda_stream)
    op = calls.op(dev)
    free = []
    for _ in range(30):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            for _ in range(8):
                calls.call(op, 0)
        calls.clear()
        g.replay()
        assert calls.right(0)
        del g
        torch.cuda.synchronize()
        free.append(torch.cuda.mem_get_info()[0])
    assert free[4] - free[-1] < 64 << 20   # 30 graphs of 8 calls, some megabytes a call if each kept its own
    dev.close()
