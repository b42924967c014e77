"""Block norm (tsn_block_norm) against the formula in 64 bits.

Tolerance of one value, from its roundings: half a unit in the last place of the result's type, and 32-bit
arithmetic on the way. A norm divides by sigma = sqrt(var + eps), so what its input is off by, at most a few
units of 2^-24 of the row's largest value (a sum of C terms pairwise adds log2 C roundings), comes out times
|w| / sigma. 64 such units cover the sums, the reciprocal root (2 ulp) and the products.
"""
import numpy as np
import pytest

import tsn

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
UNIT = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
EPS = 64 * 2.0 ** -24


@pytest.fixture(scope="module")
def dev():
    d = tsn.Device(0, stream=torch.cuda.current_stream().cuda_stream)
    yield d
    d.close()


def norm64(u, off, kind, w, b, eps):
    """(normed, bound of its 32-bit error); off: bound of u's error."""
    if kind == "none":
        return u, off
    big = u.abs().amax(-1, keepdim=True)
    mean = u.mean(-1, keepdim=True) if kind == "layer" else torch.zeros_like(big)
    sigma = ((u - mean).square().mean(-1, keepdim=True) + eps).sqrt()
    n = (u - mean) / sigma
    w = torch.ones_like(u[0, 0]) if w is None else w.double()
    err = ((off.amax(-1, keepdim=True) * 2 + EPS * big) / sigma * (1 + n.abs()) + EPS * n.abs()) * w.abs()
    n = n * w
    if b is not None:
        n = n + b.double()
        err = err + EPS * (n.abs() + b.double().abs())
    return n, err


def formula(x, y, gate, shift, scale, op, post_w=None, post_b=None, pre_w=None, pre_b=None):
    z = torch.zeros_like(x, dtype=torch.float64)
    r = op["residual_scale"]
    r = r.double() if isinstance(r, torch.Tensor) else r
    xo, off = x.double() * r, z
    if y is not None:
        n, off = norm64(y.double(), z, op["post"], post_w, post_b, op["post_eps"])
        if gate is not None:
            g = gate.double().tanh() if op["gate_tanh"] else gate.double()
            off = off * g.abs() + EPS * (n * g).abs() + (EPS * n.abs() if op["gate_tanh"] else 0)
            n = n * g
        xo = xo + n
        off = off + EPS * n.abs()
    off = off + EPS * (x.double() * r).abs()
    h, hoff = norm64(xo, off, op["pre"], pre_w, pre_b, op["pre_eps"])
    if scale is not None:
        h, hoff = h * (1 + scale.double()), hoff * (1 + scale.double()).abs() + EPS * (h * (1 + scale.double())).abs()
    if shift is not None:
        h = h + shift.double()
        hoff = hoff + EPS * (h.abs() + shift.double().abs())
    return (xo, off), (h, hoff)


def near(got, want, typ, what):
    ref, off = want
    err = (got.double() - ref).abs()
    tol = UNIT[typ] * (ref.abs() + off) + off + 1e-7 * UNIT[typ]
    tol = tol + (2.0 ** -25 if typ == "f16" else 0.0)   # half the spacing of f16 below its smallest normal
    bad = ~(err <= tol)
    assert not bool(bad.any()), (what, int(bad.sum()), float((err / tol).max()))


def make(seed, B, T, C, typ, xtyp, gate="batch", mod="batch"):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    r = lambda *s: torch.randn(s, generator=g, device="cuda")  # noqa: E731
    x, y = (r(B, T, C) * 2).to(DT[xtyp]), (r(B, T, C) * 3 + 0.5).to(DT[typ])
    shapes = {"batch": (B, 1, C), "token": (B, T, C), "one": (1, 1, C)}
    rows = lambda k: None if k == "none" else (0.3 * r(*shapes[k])).to(DT[typ])  # noqa: E731
    w = {n: 1 + 0.1 * r(C) for n in ("post_weight", "pre_weight")} | {n: 0.1 * r(C) for n in ("post_bias", "pre_bias")}
    return x, y, rows(gate), rows(mod), rows(mod), w, 1 + 0.1 * r(C)


def check_case(dev, x, y, gate, shift, scale, w, typ, xtyp, post, pre, residual_scale=1.0, gate_tanh=False, x_out=None,
               h=None, eps=1e-6):
    op = dict(post=post, pre=pre, post_eps=eps, pre_eps=eps, residual_scale=residual_scale, gate_tanh=gate_tanh)
    layer = tsn.BlockNorm(dev, x.shape[-1], **op, **w)
    want = formula(x, y, gate, shift, scale, op, w.get("post_weight"), w.get("post_bias"), w.get("pre_weight"), w.get("pre_bias"))
    x_out = torch.full_like(x, float("nan")) if x_out is None else x_out
    h = torch.full_like(y if y is not None else x, float("nan")) if h is None else h
    layer(x, y, gate=gate, shift=shift, scale=scale, x_out=x_out, h=h)
    dev.commit()
    near(x_out, want[0], xtyp, "x_out")
    near(h, want[1], typ, "h")
    return x_out, h


@pytest.mark.parametrize("typ,xtyp", [("f32", "f32"), ("f16", "f16"), ("bf16", "bf16"), ("f16", "f32"), ("bf16", "f32")])
@pytest.mark.parametrize("C", [1, 2, 7, 64, 100, 1000, 1024, 2056, 4097, 8192, 16384])
def test_widths_and_types(dev, C, typ, xtyp):
    x, y, gate, shift, scale, w, vec = make(C, 2, 5, C, typ, xtyp)
    check_case(dev, x, y, gate, shift, scale, w, typ, xtyp, "rms", "layer", residual_scale=vec)


@pytest.mark.parametrize("post", ["none", "rms", "layer"])
@pytest.mark.parametrize("pre", ["none", "rms", "layer"])
@pytest.mark.parametrize("gate,mod,tanh,r", [("none", "none", False, 1.0), ("token", "batch", True, 0.5),
                                             ("one", "token", False, "vec"), ("batch", "one", True, -0.25)])
def test_terms(dev, post, pre, gate, mod, tanh, r):
    for C, T in ((256, 33), (330, 3)):
        x, y, g, sh, sc, w, vec = make(3, 3, T, C, "bf16", "f32", gate, mod)
        check_case(dev, x, y, g, sh, sc, w, "bf16", "f32", post, pre, residual_scale=vec if r == "vec" else r, gate_tanh=tanh)
        check_case(dev, x, y, g, sh, sc, {}, "bf16", "f32", post, pre, residual_scale=vec if r == "vec" else r, gate_tanh=tanh)


@pytest.mark.parametrize("rows", [1, 2, 147, 149, 700, 5000])
@pytest.mark.parametrize("C", [64, 512, 1024, 3000])
def test_row_counts(dev, rows, C):
    x, y, g, sh, sc, w, _ = make(rows, 1, rows, C, "bf16", "bf16", "token", "batch")
    check_case(dev, x, y, g, sh, sc, w, "bf16", "bf16", "layer", "rms")


def test_first_norm_of_a_stack(dev):
    """No branch yet: h = Npre(r x); x_out is a copy, or absent."""
    x, y, _, sh, sc, w, _ = make(1, 2, 17, 192, "f16", "f16")
    check_case(dev, x, None, None, sh, sc, w, "f16", "f16", "rms", "layer")
    layer = tsn.BlockNorm(dev, 192, post="none", pre="layer")
    h = torch.empty_like(x)
    layer(x, h=h)
    dev.commit()
    near(h, norm64(x.double(), torch.zeros_like(x, dtype=torch.float64), "layer", None, None, 1e-6), "f16", "h")


def test_last_norm_of_a_stack(dev):
    """No norm after it: only x_out."""
    x, y, g, _, _, w, _ = make(2, 2, 9, 320, "bf16", "bf16")
    layer = tsn.BlockNorm(dev, 320, post="rms", pre="none", post_weight=w["post_weight"])
    out = torch.empty_like(x)
    layer(x, y, gate=g, x_out=out)
    dev.commit()
    op = dict(post="rms", pre="none", post_eps=1e-6, pre_eps=1e-6, residual_scale=1.0, gate_tanh=False)
    near(out, formula(x, y, g, None, None, op, w["post_weight"])[0], "bf16", "x_out")


@pytest.mark.parametrize("C", [256, 1000, 2048])
def test_in_place(dev, C):
    x, y, g, sh, sc, w, vec = make(4, 2, 21, C, "bf16", "f32")
    x1, h1 = check_case(dev, x, y, g, sh, sc, w, "bf16", "f32", "rms", "layer", residual_scale=vec)
    layer = tsn.BlockNorm(dev, C, post="rms", pre="layer", residual_scale=vec, **w)
    layer(x, y, gate=g, shift=sh, scale=sc, x_out=x, h=y)
    dev.commit()
    assert torch.equal(x, x1) and torch.equal(y, h1)


@pytest.mark.parametrize("pad,skip", [(8, 0), (3, 1), (1, 0), (64, 8)])
def test_strides_and_alignment(dev, pad, skip):
    """Rows inside wider rows, from any element on; time-major batches; nothing outside the rows is written."""
    B, T, C = 3, 11, 200
    x, y, g, sh, sc, w, _ = make(5, B, T, C, "f16", "f16", "token", "token")

    def inside(t, fill=None):
        wide = torch.full((T, B, C + pad + skip), float("nan") if fill is None else fill, dtype=t.dtype, device="cuda")
        view = wide[:, :, skip:skip + C].transpose(0, 1)
        view.copy_(t)
        return wide, view

    (_, xv), (_, yv), (_, gv), (_, shv), (_, scv) = map(inside, (x, y, g, sh, sc))
    wx, xo = inside(x, 7.0)
    wh, h = inside(y, 7.0)
    check_case(dev, xv, yv, gv, shv, scv, w, "f16", "f16", "rms", "layer", x_out=xo, h=h)
    for wide in (wx, wh):
        assert bool((wide[:, :, :skip] == 7.0).all()) and bool((wide[:, :, skip + C:] == 7.0).all())


def test_rows_where_a_norm_loses_digits(dev):
    """A constant row (variance 0), a zero row, and rows whose mean is far larger than their spread."""
    C = 1024
    x, y, g, sh, sc, w, _ = make(6, 1, 4, C, "f32", "f32")
    x[0, 0], y[0, 0] = 3.0, 2.0
    x[0, 1], y[0, 1] = 0.0, 0.0
    y[0, 2] += 1000.0
    x[0, 3] += 5000.0
    check_case(dev, x, y, g, sh, sc, w, "f32", "f32", "layer", "layer", eps=1e-5)


def test_not_finite_stays_in_its_row(dev):
    x, y, g, sh, sc, w, _ = make(7, 1, 6, 512, "bf16", "bf16")
    want = check_case(dev, x, y, g, sh, sc, w, "bf16", "bf16", "rms", "layer")
    x[0, 2, 5], y[0, 4, 100] = float("nan"), float("inf")
    layer = tsn.BlockNorm(dev, 512, post="rms", pre="layer", **w)
    xo, h = torch.empty_like(x), torch.empty_like(y)
    layer(x, y, gate=g, shift=sh, scale=sc, x_out=xo, h=h)
    dev.commit()
    keep = [0, 1, 3, 5]
    assert torch.equal(xo[:, keep], want[0][:, keep]) and torch.equal(h[:, keep], want[1][:, keep])
    assert bool(torch.isnan(h[0, 2]).all()) and bool(torch.isnan(h[0, 4]).all())


def test_repeats_bit_for_bit_and_on_another_stream(dev):
    x, y, g, sh, sc, w, _ = make(8, 2, 300, 1024, "bf16", "f32")
    x1, h1 = check_case(dev, x, y, g, sh, sc, w, "bf16", "f32", "rms", "layer")
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    d2 = tsn.Device(0, stream=side.cuda_stream)
    x2, h2 = check_case(d2, x, y, g, sh, sc, w, "bf16", "f32", "rms", "layer")
    side.synchronize()
    d2.close()
    assert torch.equal(x1, x2) and torch.equal(h1, h2)


def test_no_rows(dev):
    layer = tsn.BlockNorm(dev, 64)
    for shape in ((0, 5, 64), (5, 0, 64)):
        x = torch.empty(shape, device="cuda")
        layer(x, x_out=torch.empty_like(x), h=torch.empty_like(x))
    dev.commit()


def test_refusals(dev):
    x = torch.zeros(2, 3, 64, device="cuda")
    layer = tsn.BlockNorm(dev, 64)
    h = torch.empty_like(x)

    def code(call):
        with pytest.raises(tsn.TsnError) as e:
            call()
        assert "tsn_block_norm" in str(e.value)
        return e.value.code

    assert code(lambda: layer(x)) == 1                                              # no result
    assert code(lambda: layer(x, gate=x[:, :1], h=h)) == 1                          # a gate without a branch
    assert code(lambda: layer(x, h=h[:, :1].expand(2, 3, 64))) == 1                 # a result that repeats a row
    assert code(lambda: layer(x.half(), x, h=h)) == 1                               # residual narrower than the branch
    wide = torch.zeros(1, 1, 16385, device="cuda")
    assert code(lambda: tsn.BlockNorm(dev, 16385)(wide, h=torch.empty_like(wide))) == 1
    for bad in (lambda: layer(x[0], h=h), lambda: layer(x, h=h[:1]), lambda: layer(x, x, shift=x[:, :2], h=h),
                lambda: layer(x.transpose(1, 2).contiguous().transpose(1, 2), h=h), lambda: layer(x.cpu(), h=h),
                lambda: tsn.BlockNorm(dev, 64, post="batch"), lambda: tsn.BlockNorm(dev, 64, pre_weight=x)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(TypeError):
        layer(x, x, h=h.half())
    assert tsn.lib().tsn_block_norm(None, None) == 1 and tsn.lib().tsn_block_norm(dev.h, None) == 1
    a = tsn.BlockNormArgs(B=1, T=1, C=64, xtype=0, type=0, post=9, pre=0)
    assert tsn.lib().tsn_block_norm(dev.h, a) == 1
    a.post, a.type = 0, 5
    assert tsn.lib().tsn_block_norm(dev.h, a) == 1
    a.type = 0
    assert tsn.lib().tsn_block_norm(dev.h, a) == 1                                  # null x
