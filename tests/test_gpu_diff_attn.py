"""Differential attention (tsn_diff_attn) against the definition in 64 bits.

Tolerances, from the roundings: a probability is rounded to the operands' type (a share u of itself at most,
u = 2^-8 for bf16, 2^-11 for f16), its sum is the rounded ones' (off by u too), and scores, sums and products
are held in 32 bits (taken together below 2^-14 of the terms' magnitudes). So o is off by at most
E = 2.2 u sum_j (a1 + |lambda| a2)_j |v_j|, and the norm turns that into g E + |out| ||E|| / ||o||, plus half a unit
of the result. That is a bound of the worst case; as roundings fall to either side at random, the whole
result is also held to a relative 2-norm of 3 u, three times what roundings of p and of the result add up to.
"""
import math

import pytest

import tsn

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

DT = {"f16": torch.float16, "bf16": torch.bfloat16}
UNIT = {"f16": 2.0 ** -11, "bf16": 2.0 ** -8}
NAN, INF = float("nan"), float("inf")


@pytest.fixture(scope="module")
def dev():
    d = tsn.Device(0, stream=torch.cuda.current_stream().cuda_stream)
    yield d
    d.close()


def seen_of(B, Sq, Sk, lens=None, mask=None, causal=False):
    j = torch.arange(Sk, device="cuda")
    n = torch.full((B,), Sk, device="cuda") if lens is None else lens.long().clamp(0, Sk)
    seen = (j[None] < n[:, None])
    if mask is not None:
        seen = seen & (mask != 0)
    seen = seen[:, None].expand(B, Sq, Sk)
    if causal:
        i = torch.arange(Sq, device="cuda")
        seen = seen & (j[None, None] <= i[None, :, None] + n[:, None, None] - Sq)
    return seen


def formula(q, k, v, lams, lambda_init, w, eps, seen, scale=None):
    """(out, worst-case bound of its error in units u), [B, Sq, H, 2 d] in 64 bits."""
    B, Sq, H, D = q.shape
    d, G = D // 2, H // k.shape[2]
    scale = d ** -0.5 if scale is None else scale
    lam = [x.double().reshape(-1, d) for x in lams]
    lam = ((lam[0] * lam[1]).sum(-1).exp() - (lam[2] * lam[3]).sum(-1).exp() + lambda_init).expand(H)
    unseen = ~seen.any(1)[:, :, None, None]
    k, v = k.double().masked_fill(unseen, 0.0), v.double().masked_fill(unseen, 0.0)
    out, off = torch.zeros_like(q, dtype=torch.float64), torch.zeros_like(q, dtype=torch.float64)
    for h in range(H):
        o, e = 0.0, 0.0
        for part, c in ((slice(0, d), 1.0), (slice(d, D), -float(lam[h]))):
            z = scale * q[:, :, h, part].double() @ k[:, :, h // G, part].transpose(1, 2)
            z = z.masked_fill(~seen, -INF)
            a = torch.softmax(z, -1).masked_fill(~seen, 0.0)
            o = o + c * (a @ v[:, :, h // G])
            e = e + abs(c) * (a @ v[:, :, h // G].abs())
        g = (1 - lambda_init) * (w.double() if w is not None else 1.0) / (o.square().mean(-1, keepdim=True) + eps).sqrt()
        e = 2.2 * e
        out[:, :, h] = o * g
        share = e.norm(dim=-1, keepdim=True) / o.norm(dim=-1, keepdim=True).clamp(min=1e-300)
        off[:, :, h] = e * g.abs() + (o * g).abs() * (1 + share)
    return out, off


def near(got, want, typ):
    ref, off = want
    u = UNIT[typ]
    err = (got.double() - ref).abs()
    tol = off * (u + 2.0 ** -14) + (2.0 ** -24 if typ == "f16" else 1e-30)
    assert bool((err <= tol).all()), float((err / tol).nan_to_num(1e9).max())
    if float(ref.norm()):
        assert float((got.double() - ref).norm() / ref.norm()) < 3 * u


def make(seed, typ, d, B, Sq, Sk, H, Hk, gain=1.2):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    r = lambda *s: torch.randn(s, generator=g, device="cuda")  # noqa: E731
    q, k = (r(B, Sq, H, 2 * d) * gain).to(DT[typ]), (r(B, Sk, Hk, 2 * d) * gain).to(DT[typ])
    return q, k, r(B, Sk, Hk, 2 * d).to(DT[typ]), [0.1 * r(d) for _ in range(4)], 1 + 0.1 * r(2 * d)


def check_case(dev, q, k, v, lams, w, typ, lens=None, mask=None, causal=False, lambda_init=0.4, eps=1e-5, out=None, scale=None):
    B, Sq, H, D = q.shape
    seen = seen_of(B, Sq, k.shape[1], lens, mask, causal)
    want = formula(q, k, v, lams, lambda_init, w, eps, seen, scale)
    op = tsn.DiffAttention(dev, D // 2, *lams, lambda_init=lambda_init, norm_weight=w, eps=eps, scale=scale)
    out = torch.full_like(q, NAN) if out is None else out
    op(q, k, v, out, key_len=lens, key_mask=mask, causal=causal)
    dev.commit()
    near(out, want, typ)
    empty = ~seen.any(-1)
    assert bool((out[empty] == 0).all())
    return out


@pytest.mark.parametrize("typ", ["f16", "bf16"])
@pytest.mark.parametrize("d", [32, 64])
@pytest.mark.parametrize("Sq,Sk", [(1, 1), (1, 2), (1, 16), (1, 17), (1, 705), (2, 33), (4, 64), (5, 63), (16, 15), (17, 129), (100, 1),
                                   (127, 127), (128, 128), (129, 257), (1, 5000), (20, 3000), (329, 329), (300, 1500)])
def test_lengths(dev, Sq, Sk, d, typ):
    q, k, v, lams, w = make(Sq * 7 + Sk, typ, d, 2, Sq, Sk, 4, 2)
    check_case(dev, q, k, v, lams, w, typ)
    check_case(dev, q, k, v, lams, w, typ, causal=True)


@pytest.mark.parametrize("H,Hk", [(1, 1), (3, 3), (3, 1), (8, 1), (12, 4), (16, 1), (24, 3), (40, 2), (128, 1)])
@pytest.mark.parametrize("Sq", [1, 3, 50])
def test_grouped_heads(dev, H, Hk, Sq):
    q, k, v, lams, w = make(H, "bf16", 64, 1, Sq, 200, H, Hk)
    check_case(dev, q, k, v, lams, w, "bf16", causal=True)
    q, k, v, lams, w = make(H, "f16", 32, 2, Sq, 77, H, Hk)
    per_head = [x * torch.linspace(0.5, 2.0, H, device="cuda")[:, None] for x in lams]
    check_case(dev, q, k, v, per_head, w, "f16")
    check_case(dev, q, k, v, per_head, None, "f16", lambda_init=0.0)


@pytest.mark.parametrize("Sq", [1, 4, 40, 200])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("d", [32, 64])
def test_lengths_of_each_sequence(dev, Sq, causal, d):
    """Sequences of every length, none among them, shorter than their queries, past Sk and negative (clamped); what
    lies behind them is never used."""
    lens = torch.tensor([400, 0, 1, 17, 128, 129, 399, 1000, -3], dtype=torch.int32, device="cuda")
    q, k, v, lams, w = make(20 + Sq, "bf16", d, 9, Sq, 400, 4, 2)
    dead = torch.arange(400, device="cuda")[None] >= lens[:, None]
    for fill in (NAN, INF, -INF):
        k.masked_fill_(dead[:, :, None, None], fill)
        v.masked_fill_(dead[:, :, None, None], fill)
        check_case(dev, q, k, v, lams, w, "bf16", lens=lens, causal=causal)


@pytest.mark.parametrize("Sq", [1, 5, 60, 300])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("typ,d", [("bf16", 64), ("f16", 32)])
def test_masked_keys(dev, Sq, causal, typ, d):
    """Holes, a masked start, a masked end, one key only, and no key at all; masked keys hold NaN and infinities."""
    Sk = 330
    q, k, v, lams, w = make(30 + Sq, typ, d, 6, Sq, Sk, 4, 4)
    mask = torch.ones(6, Sk, dtype=torch.uint8, device="cuda")
    mask[0, ::3] = 0
    mask[1, :200] = 0
    mask[2, 131:] = 0
    mask[3] = 0
    mask[3, 150] = 255
    mask[4] = 0
    hidden = mask == 0
    k0, v0 = k.clone(), v.clone()
    for fill in (NAN, INF, -INF, torch.finfo(DT[typ]).min):
        k.masked_fill_(hidden[:, :, None, None], fill)
        v.masked_fill_(hidden[:, :, None, None], fill)
        check_case(dev, q, k, v, lams, w, typ, mask=mask, causal=causal)
    one = mask[:1].bool()
    lens = torch.tensor([330, 300, 2, 0, 128, 129], dtype=torch.int32, device="cuda")
    check_case(dev, q, k0, v0, lams, w, typ, mask=one, lens=lens, causal=causal)   # one mask for the batch, with lengths


@pytest.mark.parametrize("Sq,Sk", [(4, 40), (16, 700), (200, 200), (129, 513)])
@pytest.mark.parametrize("fill", [NAN, INF])
def test_not_finite_keys_of_the_future(dev, Sq, Sk, fill):
    """A causal row is not touched by what later keys and values hold; rows that see such a value are NaN."""
    q, k, v, lams, w = make(40, "bf16", 64, 2, Sq, Sk, 4, 2)
    clean = check_case(dev, q, k, v, lams, w, "bf16", causal=True)
    at = Sk - Sq // 2 - 1
    k[:, at + 1:, :, 3] = fill
    v[:, at + 1:, :, ::7] = fill
    op = tsn.DiffAttention(dev, 64, *lams, lambda_init=0.4, norm_weight=w, eps=1e-5)
    out = torch.empty_like(q)
    op(q, k, v, out, causal=True)
    dev.commit()
    first = at + 1 - (Sk - Sq)   # the first row that sees a changed key
    assert torch.equal(out[:, :first], clean[:, :first])
    assert bool(torch.isnan(out[:, first:]).all())


@pytest.mark.parametrize("Sq", [1, 64])
def test_not_finite_value_in_sight(dev, Sq):
    for fill in (NAN, INF, -INF):
        q, k, v, lams, w = make(41, "f16", 64, 1, Sq, 100, 2, 2)
        clean = check_case(dev, q, k, v, lams, w, "f16")
        v[0, 30, 1, 5] = fill
        op = tsn.DiffAttention(dev, 64, *lams, lambda_init=0.4, norm_weight=w, eps=1e-5)
        out = torch.empty_like(q)
        op(q, k, v, out)
        dev.commit()
        assert torch.equal(out[:, :, 0], clean[:, :, 0]) and bool(torch.isnan(out[:, :, 1]).all())


@pytest.mark.parametrize("Sq", [1, 150])
@pytest.mark.parametrize("typ", ["f16", "bf16"])
def test_scores_of_every_size(dev, Sq, typ):
    """Maximum first, last, everywhere the same, and rising along the keys; scores far beyond what exp holds."""
    q, k, v, lams, w = make(50, typ, 64, 6, Sq, 1000, 2, 2)
    q[:] = q.abs()
    k[0, 0], k[1, 999] = 12.0, 12.0
    k[2] = 0.25
    k[3] = (torch.linspace(0, 6, 1000, device="cuda")[:, None, None]).to(k.dtype)
    k[4] = (torch.linspace(6, -6, 1000, device="cuda")[:, None, None]).to(k.dtype)
    k[5] = -20.0
    v += 0.5
    check_case(dev, q, k, v, lams, w, typ)
    check_case(dev, q, k, v, lams, w, typ, scale=3.0)


def test_orders_and_strides(dev):
    """Slices of a packed projection; head-major caches longer than the sequence; a batch that shares its keys."""
    B, Sq, Sk, H, Hk, D = 2, 70, 90, 4, 2, 128
    for Sq in (1, 70):
        q, k, v, lams, w = make(60, "bf16", 64, B, Sq, Sk, H, Hk)
        want = check_case(dev, q, k, v, lams, w, "bf16", causal=True)
        packed = torch.zeros(B, Sq, (H + 1) * D, dtype=torch.bfloat16, device="cuda")
        packed[..., D:].view(B, Sq, H, D).copy_(q)
        cache = torch.full((2, B, Hk, 200, D), NAN, dtype=torch.bfloat16, device="cuda")
        kc, vc = (cache[i, :, :, 30:30 + Sk].transpose(1, 2) for i in (0, 1))
        kc.copy_(k)
        vc.copy_(v)
        wide = torch.full((B, H, Sq, D + 8), 7.0, dtype=torch.bfloat16, device="cuda")
        out = wide[..., :D].transpose(1, 2)
        got = check_case(dev, packed[..., D:].unflatten(-1, (H, D)), kc, vc, lams, w, "bf16", causal=True, out=out)
        assert torch.equal(got, want) and bool((wide[..., D:] == 7.0).all())
        shared = check_case(dev, q, k[:1].expand(B, -1, -1, -1), v[:1].expand(B, -1, -1, -1), lams, w, "bf16")
        assert torch.equal(shared[0], check_case(dev, q[:1], k[:1], v[:1], lams, w, "bf16")[0])


@pytest.mark.parametrize("Sq", [1, 40])
def test_offsets_past_32_bits(dev, Sq):
    """Caches whose sequences lie more than 2^31 elements apart."""
    far = 2 ** 31 + 64
    store = torch.empty(far + 2 ** 18, dtype=torch.float16, device="cuda")
    q, k, v, lams, w = make(70, "f16", 64, 2, Sq, 300, 2, 2)
    kv = store.as_strided((2, 300, 2, 2, 128), (far, 512, 256, 128, 1))
    kv[:, :, :, 0].copy_(k)
    kv[:, :, :, 1].copy_(v)
    check_case(dev, q, kv[:, :, :, 0], kv[:, :, :, 1], lams, w, "f16", causal=True)


@pytest.mark.parametrize("Sq,Sk,H,Hk", [(1, 20000, 8, 2), (3, 9000, 5, 5), (64, 6000, 2, 1), (600, 900, 4, 4)])
def test_repeats_bit_for_bit(dev, Sq, Sk, H, Hk):
    q, k, v, lams, w = make(80, "bf16", 64, 1, Sq, Sk, H, Hk)
    lens = torch.tensor([Sk - 5], dtype=torch.int32, device="cuda")
    op = tsn.DiffAttention(dev, 64, *lams, lambda_init=0.4, norm_weight=w)
    outs = []
    for _ in range(8):
        outs.append(torch.empty_like(q))
        op(q, k, v, outs[-1], key_len=lens, causal=True)
    dev.commit()
    assert all(torch.equal(outs[0], o) for o in outs[1:])


def test_streams_share_a_device_handle(dev):
    """Calls that split their keys, on streams in turn, share the handle's workspace in the order of the calls."""
    q, k, v, lams, w = make(81, "bf16", 64, 1, 2, 30000, 8, 8)
    q2 = (q.float() * -1.0).to(q.dtype)
    op = tsn.DiffAttention(dev, 64, *lams, lambda_init=0.4, norm_weight=w)
    want = [torch.empty_like(q) for _ in range(2)]
    op(q, k, v, want[0])
    op(q2, k, v, want[1])
    dev.commit()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[torch.empty_like(q) for _ in range(2)] for _ in range(10)]
    for pair in got:
        for s, x, o in zip(streams, (q, q2), pair):
            tsn.check(tsn.lib().tsn_device_set_stream(dev.h, s.cuda_stream))
            op(x, k, v, o)
    torch.cuda.synchronize()
    tsn.check(tsn.lib().tsn_device_set_stream(dev.h, torch.cuda.current_stream().cuda_stream))
    assert all(torch.equal(a, b) for pair in got for a, b in zip(pair, want))


@pytest.mark.parametrize("Sq,Sk", [(1, 8000), (260, 260)])
def test_in_a_cuda_graph(dev, Sq, Sk):
    q, k, v, lams, w = make(82, "bf16", 64, 1, Sq, Sk, 4, 4)
    op = tsn.DiffAttention(dev, 64, *lams, lambda_init=0.4, norm_weight=w)
    out, want = torch.empty_like(q), torch.empty_like(q)
    side = torch.cuda.Stream()
    d2 = tsn.Device(0, stream=side.cuda_stream)
    op2 = tsn.DiffAttention(d2, 64, *lams, lambda_init=0.4, norm_weight=w)
    with torch.cuda.stream(side):
        op2(q, k, v, out)
    side.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        op2(q, k, v, out)
    for sign in (1.0, -1.0):
        q.copy_(q.float() * sign)
        op(q, k, v, want)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
    del g
    d2.close()


def test_nothing_to_do(dev):
    q, k, v, lams, w = make(90, "bf16", 64, 2, 3, 4, 2, 2)
    out = torch.full_like(q, NAN)
    op = tsn.DiffAttention(dev, 64, *lams, lambda_init=0.4, norm_weight=w)
    op(q, k[:, :0], v[:, :0], out)   # no keys: every row is empty
    dev.commit()
    assert bool((out == 0).all())
    op(q[:, :0], k, v, out[:, :0])
    op(q[:0], k[:0], v[:0], out[:0])
    dev.commit()


def test_refusals(dev):
    q, k, v, lams, w = make(91, "bf16", 64, 2, 3, 4, 4, 2)
    out = torch.empty_like(q)
    op = tsn.DiffAttention(dev, 64, *lams, lambda_init=0.4, norm_weight=w)

    def code(call):
        with pytest.raises(tsn.TsnError) as e:
            call()
        assert "tsn_diff_attn" in str(e.value)
        return e.value.code

    assert code(lambda: op(q.float(), k.float(), v.float(), out.float())) == 1
    assert code(lambda: op(q[:, :, :3], k, v, out[:, :, :3])) == 1                            # 3 heads over 2
    assert code(lambda: op(q, k, v, out[:, :1].expand(2, 3, 4, 128))) == 1
    big = torch.zeros(2, 4, 2, 136, dtype=torch.bfloat16, device="cuda")
    assert code(lambda: op(q, big[..., 4:132], v, out)) == 1                                  # 8 bytes off
    odd = torch.zeros(2, 4, 2, 132, dtype=torch.bfloat16, device="cuda")
    assert code(lambda: op(q, odd[..., :128], v, out)) == 1                                   # rows of 264 bytes
    l48 = [x[:48].contiguous() for x in lams]
    x = torch.zeros(1, 1, 1, 96, dtype=torch.bfloat16, device="cuda")
    assert code(lambda: tsn.DiffAttention(dev, 48, *l48, lambda_init=0.4)(x, x, x, x.clone())) == 1
    x = torch.zeros(1, 1, 129, 128, dtype=torch.bfloat16, device="cuda")
    assert code(lambda: op(x, x[:, :, :1], x[:, :, :1], x.clone())) == 1                      # 129 heads over one
    assert code(lambda: tsn.DiffAttention(dev, 64, *lams, lambda_init=0.4, scale=-1.0)(q, k, v, out)) == 1
    assert code(lambda: tsn.DiffAttention(dev, 64, *lams, lambda_init=0.4, eps=NAN)(q, k, v, out)) == 1
    lens, mask = torch.zeros(2, dtype=torch.int32, device="cuda"), torch.ones(2, 4, dtype=torch.uint8, device="cuda")
    for bad in (lambda: op(q[..., :64], k, v, out), lambda: op(q, k[..., :64], v, out), lambda: op(q, k, v[:, :3], out),
                lambda: op(q, k, v, out[:1]), lambda: op(q, k, v, out, key_len=lens.long()),
                lambda: op(q, k, v, out, key_len=lens[:1]), lambda: op(q, k, v, out, key_mask=mask[:, :3]),
                lambda: op(q, k, v, out, key_mask=mask.float()), lambda: op(q, k.cpu(), v, out),
                lambda: tsn.DiffAttention(dev, 64, *[x[:32] for x in lams], lambda_init=0.4),
                lambda: tsn.DiffAttention(dev, 64, *lams, lambda_init=0.4, norm_weight=w[:64]),
                lambda: tsn.DiffAttention(dev, 64, *[x.expand(3, 64) for x in lams], lambda_init=0.4)(q, k, v, out)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(TypeError):
        op(q, k.half(), v, out)
    assert tsn.lib().tsn_diff_attn(None, None) == 1 and tsn.lib().tsn_diff_attn(dev.h, None) == 1
    assert tsn.lib().tsn_diff_attn(dev.h, tsn.DiffAttnArgs(B=1, Sq=1, Sk=1, H=1, Hk=1, d=64, type=2)) == 1   # null operands
