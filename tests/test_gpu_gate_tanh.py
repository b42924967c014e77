"""tanh gates of the block norm (tsn_block_norm) at every magnitude, with nothing beside the branch that could hide an error.

Tolerance, relative to each value: the norm's sum of squares, reciprocal root and products stay below 32 units of 2^-24
(a sum of squares has no cancellation: log2 C roundings of its parts, then 2 ulp and three products), the gate's tanh below
another 32; then half a unit of the result's type. The norm after it sees those 64 units in each value and in the row's
root mean square, and adds 32 of its own: 160.
"""
import pytest

import tsn

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
HALF = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
LEAST = {"f32": 2.0 ** -126, "f16": 2.0 ** -25, "bf16": 2.0 ** -126}   # below the normal values: half their spacing, or flushed


@pytest.fixture(scope="module")
def dev():
    d = tsn.Device(0, stream=torch.cuda.current_stream().cuda_stream)
    yield d
    d.close()


@pytest.mark.parametrize("typ,xtyp", [("f32", "f32"), ("f16", "f16"), ("bf16", "bf16"), ("f16", "f32"), ("bf16", "f32")])
@pytest.mark.parametrize("C", [128, 1021, 1022, 1024, 4096, 9000])
def test_gates_of_every_size(dev, C, typ, xtyp):
    rows = 81
    g = torch.Generator(device="cuda")
    g.manual_seed(C)
    r = lambda *s: torch.randn(s, generator=g, device="cuda")  # noqa: E731
    size = 10.0 ** torch.linspace(-7, 1.2, rows, device="cuda")[None, :, None]
    gate = (size * (0.5 + 0.5 * torch.rand(1, rows, C, generator=g, device="cuda")) * r(1, rows, C).sign()).to(DT[typ])
    y, x = r(1, rows, C).to(DT[typ]), r(1, rows, C).to(DT[xtyp])
    w, eps = 1 + 0.1 * r(C), 1e-24
    op = tsn.BlockNorm(dev, C, post="rms", pre="rms", post_weight=w, post_eps=eps, pre_eps=eps, residual_scale=0.0, gate_tanh=True)
    x_out, h = torch.empty_like(x), torch.empty_like(y)
    op(x, y, gate=gate, x_out=x_out, h=h)
    dev.commit()
    rms = lambda u: u / (u.square().mean(-1, keepdim=True) + eps).sqrt()  # noqa: E731
    want = gate.double().tanh() * rms(y.double()) * w.double()
    for got, ref, t, units in ((x_out, want, xtyp, 64), (h, rms(want), typ, 160)):
        tol = ref.abs() * (units * 2.0 ** -24 + HALF[t]) + LEAST[t]
        err = (got.double() - ref).abs()
        assert bool((err <= tol).all()), float((err / tol).max())


@pytest.mark.parametrize("typ", ["f32", "f16", "bf16"])
def test_gates_that_are_zero_infinite_or_nan(dev, typ):
    y, x = torch.ones(1, 1, 64, device="cuda").to(DT[typ]), torch.zeros(1, 1, 64, device="cuda").to(DT[typ])
    gate = torch.zeros_like(y)
    gate[0, 0, 1], gate[0, 0, 2], gate[0, 0, 3], gate[0, 0, 4], gate[0, 0, 5] = float("inf"), -float("inf"), float("nan"), 60000.0, -60000.0
    op = tsn.BlockNorm(dev, 64, post="none", pre="none", gate_tanh=True)
    out = torch.empty_like(x)
    op(x, y, gate=gate, x_out=out)
    dev.commit()
    got = out[0, 0].float().tolist()
    assert got[0] == 0.0 and got[1] == got[4] == 1.0 and got[2] == got[5] == -1.0 and got[3] != got[3] and not any(got[6:])
