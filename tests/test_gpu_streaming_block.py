"""The example block that runs the transformer-block operators together: chunks of any size give what all tokens at once
give, and both what the formulas give in 64 bits.

Tolerance: queries, keys, values and attention results are rounded to float16 (half a unit 2^-11 each), which passes through
two norms and two projections of random weights (gain about one); four such roundings with the maps' own stay
below 2^-9 of the block's result.
"""
import os
import sys

import pytest

import tsn

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))


@pytest.fixture(scope="module")
def dev():
    d = tsn.Device(0, stream=torch.cuda.current_stream().cuda_stream)
    yield d
    d.close()


def reference(frames, height, width, seed, dev):
    """The block's formulas in 64 bits on the example's weights and inputs."""
    import streaming_block as ex
    b = ex.StreamingBlock(dev, cache=1, seed=seed)
    g = torch.Generator(device="cuda")
    g.manual_seed(seed + 1)
    n = frames * height * width
    x = torch.randn(b.B, n, b.C, generator=g, device="cuda").double()
    pos = ex.positions(frames, height, width).double()
    rms = lambda u, w, eps=1e-6: u / torch.sqrt(u.square().mean(-1, keepdim=True) + eps) * w.double()  # noqa: E731
    lin = lambda u, w: u @ w.double().T  # noqa: E731
    h = rms(x, b.first._keep[2]) * (1 + b.scale1.double()) + b.shift1.double()

    def turned(u, w):
        u = rms(u, w)
        y = u.clone()
        j = 0
        for axis, pairs in enumerate((8, 12, 12)):
            for i in range(pairs):
                t = pos[:, axis] * 10000.0 ** (-i / pairs)
                c, s = t.cos()[None, :, None], t.sin()[None, :, None]
                y[..., 2 * j] = u[..., 2 * j] * c - u[..., 2 * j + 1] * s
                y[..., 2 * j + 1] = u[..., 2 * j] * s + u[..., 2 * j + 1] * c
                j += 1
        return y

    d, H, Hk = b.d, b.H, b.Hk
    q = turned(lin(h, b.wq).view(b.B, n, 2 * H, d), b.rope._keep[0])
    k = turned(lin(h, b.wk).view(b.B, n, 2 * Hk, d), b.rope._keep[1])
    v = lin(h, b.wv).view(b.B, n, Hk, 2 * d)
    lams = [t.double() for t in b.attention._keep[:4]]
    lam = torch.exp(lams[0] @ lams[1]) - torch.exp(lams[2] @ lams[3]) + 0.4
    late = torch.triu(torch.ones(n, n, dtype=torch.bool, device="cuda"), 1)
    o = torch.empty(b.B, n, H, 2 * d, dtype=torch.float64, device="cuda")
    for head in range(H):
        kv = head // (H // Hk)
        maps = [torch.softmax((q[:, :, 2 * head + m] @ k[:, :, 2 * kv + m].transpose(1, 2) * d ** -0.5).masked_fill(late, float("-inf")), -1)
                for m in (0, 1)]
        o[:, :, head] = rms((maps[0] - lam * maps[1]) @ v[:, :, kv], b.attention._keep[4], 1e-5) * 0.6
    y = lin(o.view(b.B, n, -1), b.wo)
    x1 = 0.9 * x + b.gate1.double().tanh() * rms(y, b.middle._keep[0])
    h = rms(x1, b.middle._keep[2]) * (1 + b.scale2.double()) + b.shift2.double()
    y = lin(torch.nn.functional.silu(lin(h, b.w1)), b.w2)
    return 0.9 * x1 + b.gate2.double().tanh() * rms(y, b.last._keep[0])


def test_chunks_agree_with_all_tokens_and_the_formulas(dev):
    import streaming_block as ex
    size = (5, 3, 7)
    want = reference(*size, 3, dev)
    for chunk in (105, 40, 17, 1):
        got = ex.run(dev, *size, chunk, seed=3)
        dev.commit()
        assert float((got.double() - want).norm() / want.norm()) < 2.0 ** -9, chunk


def test_a_full_cache_is_refused(dev):
    import streaming_block as ex
    b = ex.StreamingBlock(dev, cache=4)
    with pytest.raises(ValueError):
        b(torch.zeros(b.B, 5, b.C, device="cuda"), ex.positions(5, 1, 1))
