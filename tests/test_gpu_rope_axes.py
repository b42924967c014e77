"""Rotary positions with several axes (tsn_rope_axes) against the formula in 64 bits.

Tolerance of one value, from its roundings: half a unit in the last place of the result's type; the angle's
cosine and sine, off by at most 2^-22 (an angle held to 2^-25 of a turn, sincospi to 2 ulp); and 32-bit
products and norm, 16 units of 2^-24 of the head's values.
"""
import math

import numpy as np
import pytest

import tsn

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
UNIT = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}


@pytest.fixture(scope="module")
def dev():
    d = tsn.Device(0, stream=torch.cuda.current_stream().cuda_stream)
    yield d
    d.close()


def formula(x, pos, pairs, theta, scale, layout, w, eps):
    """x [B, S, H, D], pos [B, S, A] -> (result, largest value of each pair for the bound)."""
    x = x.double()
    if w is not None:
        x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + eps) * w.double()
    P = sum(pairs)
    y, j = x.clone(), 0
    big = x.abs().clone()
    for a, n in enumerate(pairs):
        for i in range(n):
            f = scale[a] * theta[a] ** (-i / n) / (2 * math.pi)
            t = (pos[..., a].double() * f).remainder(1.0) * (2 * math.pi)
            c, s = t.cos()[:, :, None], t.sin()[:, :, None]
            e0, e1 = (j, j + P) if layout == "half" else (2 * j, 2 * j + 1)
            u, v = x[..., e0], x[..., e1]
            y[..., e0], y[..., e1] = u * c - v * s, u * s + v * c
            big[..., e0] = big[..., e1] = u.abs() + v.abs()
            j += 1
    return y, big


def near(got, want, typ, what):
    ref, big = want
    tol = UNIT[typ] * (ref.abs() + big * 2.0 ** -20) + big * (2.0 ** -22 + 16 * 2.0 ** -24) + (2.0 ** -25 if typ == "f16" else 1e-30)
    err = (got.double() - ref).abs()
    assert bool((err <= tol).all()), (what, float((err / tol).max()))


def make(seed, B, S, Hq, Hk, D, typ):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    r = lambda *s: torch.randn(s, generator=g, device="cuda")  # noqa: E731
    return r(B, S, Hq, D).to(DT[typ]), r(B, S, Hk, D).to(DT[typ]), 1 + 0.2 * r(D), 1 + 0.2 * r(D)


def check_case(dev, q, k, pos, pairs, typ, layout="interleaved", theta=10000.0, scale=1.0, qw=None, kw=None, eps=1e-6,
               q_out=None, k_out=None):
    n = len(pairs)
    th = [theta] * n if isinstance(theta, float) else theta
    sc = [scale] * n if isinstance(scale, float) else scale
    D = (q if q is not None else k).shape[-1]
    full = pos if pos.dim() == 3 else pos[None]
    full = full.expand((q if q is not None else k).shape[0], -1, -1)
    want = [None if x is None else formula(x, full, pairs, th, sc, layout, w, eps) for x, w in ((q, qw), (k, kw))]
    op = tsn.RopeAxes(dev, D, pairs, theta=theta, scale=scale, layout=layout, q_norm=qw, k_norm=kw, eps=eps)
    outs = [o if o is not None else None if x is None else torch.full_like(x, float("nan")) for x, o in ((q, q_out), (k, k_out))]
    op(q, k, pos, *outs)
    dev.commit()
    for o, w, name in zip(outs, want, "qk"):
        if w is not None:
            near(o, w, typ, name)
    return outs


def grid(T, Y, X, start=0):
    g = torch.stack(torch.meshgrid(torch.arange(T), torch.arange(Y), torch.arange(X), indexing="ij"), -1).reshape(-1, 3)
    return (g + torch.tensor([start, 0, 0])).to(torch.int32).cuda()


@pytest.mark.parametrize("typ", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("layout", ["interleaved", "half"])
@pytest.mark.parametrize("D,pairs", [(64, (8, 12, 12)), (128, (16, 24, 24)), (32, (4, 6, 6)), (64, (32,)), (64, (8, 4, 4)),
                                     (96, (20, 14, 11)), (80, (13, 13, 14)), (256, (40, 44, 44)), (2, (1,)), (6, (1, 1, 1)),
                                     (64, (5, 0, 7, 9)), (64, (0, 0))])
def test_heads_and_axes(dev, D, pairs, layout, typ):
    q, k, qw, kw = make(D, 2, 30, 5, 3, D, typ)
    pos = grid(5, 2, 3)[:, [0, 1, 2, 0][: len(pairs)]].contiguous()
    check_case(dev, q, k, pos, pairs, typ, layout, qw=qw, kw=kw)
    check_case(dev, q, k, pos, pairs, typ, layout)


@pytest.mark.parametrize("B,S,Hq,Hk", [(1, 1, 1, 1), (1, 1, 16, 16), (8, 1, 32, 4), (1, 2, 3, 1), (3, 77, 16, 2), (1, 1021, 7, 7),
                                       (2, 2100, 4, 4)])
def test_sizes(dev, B, S, Hq, Hk):
    q, k, qw, kw = make(S, B, S, Hq, Hk, 64, "bf16")
    pos = torch.stack((torch.arange(S) // 7, torch.arange(S) % 7, torch.arange(S) % 5), -1).to(torch.int32).cuda()
    check_case(dev, q, k, pos, (12, 10, 10), "bf16", qw=qw)   # only the queries are normed
    check_case(dev, q, k, pos, (12, 10, 10), "bf16", "half", kw=kw)


def test_far_and_negative_positions_keep_their_precision(dev):
    """Positions up to the ends of 32 bits, one list of positions per sequence."""
    q, k, qw, kw = make(9, 4, 64, 2, 2, 64, "f32")
    pos = torch.randint(-2 ** 31, 2 ** 31 - 1, (4, 64, 2), generator=torch.Generator().manual_seed(0), dtype=torch.int64)
    pos[0, 0], pos[0, 1], pos[0, 2] = -2 ** 31, 2 ** 31 - 1, -1
    check_case(dev, q, k, pos.to(torch.int32).cuda() // 4096, (16, 16), "f32", qw=qw, kw=kw)
    check_case(dev, q, k, torch.full((4, 64, 2), -3, dtype=torch.int32, device="cuda"), (16, 16), "f32")


def test_angle_at_the_ends_of_32_bits(dev):
    """The whole product of position and fraction, in Python's integers."""
    pos = torch.tensor([[-2 ** 31], [2 ** 31 - 1], [123456789], [-987654321]], dtype=torch.int32, device="cuda")
    op = tsn.RopeAxes(dev, 64, (32,))
    q = torch.zeros(1, 4, 1, 64, device="cuda")
    q[..., 0::2] = 1.0
    out = torch.empty_like(q)
    op(q, None, pos, out)
    dev.commit()
    for s in range(4):
        for j in range(32):
            part = (int(pos[s, 0]) * op._plan.turn[j]) % 2 ** 64
            a = 2 * math.pi * (part / 2.0 ** 64)
            assert abs(float(out[0, s, 0, 2 * j]) - math.cos(a)) < 2 ** -21
            assert abs(float(out[0, s, 0, 2 * j + 1]) - math.sin(a)) < 2 ** -21
    assert op._plan.turn[0] == int(1.0 / (2 * math.pi) * 2.0 ** 64)


@pytest.mark.parametrize("typ", ["f32", "bf16"])
def test_bases_and_scales_of_each_axis(dev, typ):
    q, k, _, _ = make(10, 2, 40, 3, 3, 64, typ)
    pos = torch.randint(0, 50, (2, 40, 3), dtype=torch.int32, device="cuda")
    outs = check_case(dev, q, k, pos, (10, 11, 11), typ, theta=[100.0, 1e4, 5e5], scale=[0.25, 1.0, 7.5])
    # a negative scale turns back
    back = check_case(dev, outs[0], outs[1], pos, (10, 11, 11), typ, theta=[100.0, 1e4, 5e5], scale=[-0.25, -1.0, -7.5])
    assert float((back[0].float() - q.float()).abs().max()) < (0.05 if typ == "bf16" else 1e-5)


def test_one_of_the_two_and_in_place(dev):
    q, k, qw, kw = make(11, 2, 50, 6, 2, 64, "bf16")
    pos = grid(2, 5, 5)
    a, b = check_case(dev, q, k, pos, (10, 10, 12), "bf16", qw=qw, kw=kw)
    a1, _ = check_case(dev, q, None, pos, (10, 10, 12), "bf16", qw=qw)
    _, b1 = check_case(dev, None, k, pos, (10, 10, 12), "bf16", kw=kw)
    op = tsn.RopeAxes(dev, 64, (10, 10, 12), q_norm=qw, k_norm=kw)
    op(q, k, pos)
    dev.commit()
    assert torch.equal(a, a1) and torch.equal(b, b1) and torch.equal(a, q) and torch.equal(b, k)


@pytest.mark.parametrize("layout", ["interleaved", "half"])
@pytest.mark.parametrize("skip", [0, 1, 2, 8])
def test_strides_orders_and_alignment(dev, skip, layout):
    """Slices of a packed projection in; head-major rows of a longer cache, from an odd element on, out."""
    B, S, Hq, Hk, D = 2, 23, 4, 2, 64
    q, k, qw, kw = make(12, B, S, Hq, Hk, D, "f16")
    wide = torch.randn(B, S, (Hq + 2 * Hk) * D + 2 * skip, device="cuda").half()
    qs = wide[..., skip: skip + Hq * D].unflatten(-1, (Hq, D))
    ks = wide[..., skip + Hq * D: skip + (Hq + Hk) * D].unflatten(-1, (Hk, D))
    cache = torch.full((B, Hk, 100, D + 8), 7.0, dtype=torch.float16, device="cuda")
    kc = cache[:, :, 40:40 + S, skip % 8: skip % 8 + D].transpose(1, 2)
    qo = torch.full((B, Hq, S, D), float("nan"), dtype=torch.float16, device="cuda").transpose(1, 2)
    pos = torch.randint(0, 99, (S, 2), dtype=torch.int32, device="cuda")
    check_case(dev, qs, ks, pos, (15, 17), "f16", layout, qw=qw, kw=kw, q_out=qo, k_out=kc)
    rest = torch.ones_like(cache, dtype=torch.bool)
    rest[:, :, 40:40 + S, skip % 8: skip % 8 + D] = False
    assert bool((cache[rest] == 7.0).all())


def test_offsets_past_32_bits(dev):
    """A batch stride of more than 2^31 elements."""
    far = 2 ** 31 + 64
    store = torch.empty(far + 4096, dtype=torch.bfloat16, device="cuda")
    q = store.as_strided((2, 8, 4, 64), (far, 256, 64, 1))
    q.copy_(torch.randn(2, 8, 4, 64, device="cuda"))
    check_case(dev, q, None, grid(2, 2, 2), (10, 10, 12), "bf16", q_out=torch.empty(2, 8, 4, 64, dtype=torch.bfloat16, device="cuda"))


def test_not_finite_stays_in_its_head(dev):
    q, k, qw, kw = make(13, 1, 9, 4, 4, 64, "bf16")
    want = check_case(dev, q, k, grid(1, 3, 3), (10, 10, 12), "bf16", qw=qw, kw=kw)
    q[0, 4, 2, 10] = float("nan")
    op = tsn.RopeAxes(dev, 64, (10, 10, 12), q_norm=qw, k_norm=kw)
    op(q, k, grid(1, 3, 3))
    dev.commit()
    assert bool(torch.isnan(q[0, 4, 2]).all()) and torch.equal(k, want[1])
    q[0, 4, 2] = want[0][0, 4, 2]
    assert torch.equal(q, want[0])


def test_no_tokens_or_heads(dev):
    op = tsn.RopeAxes(dev, 64, (32,))
    q = torch.empty(2, 0, 4, 64, device="cuda")
    op(q, q, torch.empty(0, 1, dtype=torch.int32, device="cuda"))
    q = torch.empty(0, 3, 4, 64, device="cuda")
    op(q, q, torch.zeros(3, 1, dtype=torch.int32, device="cuda"))
    dev.commit()


def test_refusals(dev):
    def code(call, what):
        with pytest.raises(tsn.TsnError) as e:
            call()
        assert what in str(e.value)
        return e.value.code

    for make_plan in (lambda: tsn.RopeAxes(dev, 63, (8,)), lambda: tsn.RopeAxes(dev, 258, (8,)), lambda: tsn.RopeAxes(dev, 64, ()),
                      lambda: tsn.RopeAxes(dev, 64, (1,) * 5), lambda: tsn.RopeAxes(dev, 64, (20, 13)),
                      lambda: tsn.RopeAxes(dev, 64, (8,), theta=0.0), lambda: tsn.RopeAxes(dev, 64, (8,), scale=float("inf")),
                      lambda: tsn.RopeAxes(dev, 64, (8,), theta=float("nan"))):
        assert code(make_plan, "tsn_rope_plan") == 1
    op = tsn.RopeAxes(dev, 64, (16, 16))
    q = torch.zeros(2, 3, 4, 64, device="cuda")
    pos = torch.zeros(3, 2, dtype=torch.int32, device="cuda")
    assert code(lambda: op(q, None, pos, q[:, :1].expand(2, 3, 4, 64)), "tsn_rope_axes") == 1
    for bad in (lambda: op(q, None, pos.long()), lambda: op(q, None, pos[:2]), lambda: op(q, None, pos[:, :1]),
                lambda: op(q[..., :32], None, pos), lambda: op(q, q[:1], pos), lambda: op(q, None, pos.cpu()),
                lambda: op(q, None, pos, q[:1]), lambda: tsn.RopeAxes(dev, 64, (8,), layout="other"),
                lambda: tsn.RopeAxes(dev, 64, (8, 8), theta=(1e4,)), lambda: tsn.RopeAxes(dev, 64, (8,), q_norm=pos)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(TypeError):
        op(q, q.half(), pos)
    with pytest.raises(TypeError):
        op(q.double(), None, pos)
    broken = tsn.RopePlan(D=64, axes=1, P=40)
    args = tsn.RopeArgs(B=1, S=1, Hq=1)
    assert tsn.lib().tsn_rope_axes(dev.h, broken, args) == 1
    assert tsn.lib().tsn_rope_axes(dev.h, None, args) == 1
    assert tsn.lib().tsn_rope_axes(None, broken, args) == 1
