"""A device handle whose call was captured in a CUDA graph while no work was pending commits as before: a captured call is no
work of the handle's until the graph is replayed, and leaves its timing events alone."""
import pytest
import torch

import tsn

pytestmark = pytest.mark.gpu


def calls(dev):
    """One call of each operator, as closures over their own tensors, and their results."""
    r = lambda *s: torch.randn(s, device="cuda")  # noqa: E731
    x, y, h = r(2, 3, 64), r(2, 3, 64), torch.empty(2, 3, 64, device="cuda")
    norm = tsn.BlockNorm(dev, 64, post="rms", pre="rms")
    q, out, pos = r(1, 4, 2, 32), torch.empty(1, 4, 2, 32, device="cuda"), torch.arange(4, dtype=torch.int32, device="cuda")[:, None]
    rope = tsn.RopeAxes(dev, 32, (16,))
    a, k, v = (r(1, s, 2, 64).half() for s in (2, 9, 9))
    o = torch.empty_like(a)
    attn = tsn.DiffAttention(dev, 32, *(0.1 * r(32) for _ in range(4)), lambda_init=0.3)
    return [(lambda: norm(x, y, h=h), h), (lambda: rope(q, None, pos, q_out=out), out), (lambda: attn(a, k, v, o), o)]


@pytest.mark.parametrize("which", range(3))
def test_commit_after_capture(which):
    side = torch.cuda.Stream()
    dev = tsn.Device(0, stream=side.cuda_stream)
    call, result = calls(dev)[which]
    torch.cuda.synchronize()
    call()
    dev.commit()
    want = result.clone()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        call()
    dev.commit()            # nothing is pending
    result.zero_()
    torch.cuda.synchronize()
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(result, want)
    call()
    dev.commit()            # this call's time, not the capture's
    assert 0.0 < tsn.lib().tsn_last_gpu_ms(dev.h) < 1e3
    del g
    dev.close()
