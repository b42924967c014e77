"""Differential attention whose keys are split over the workspace: calls that run at the same time on streams that
share a handle never share their sums."""
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
