"""Cases that measure the transformer-block operators: block norm, rotary positions with several axes,
differential attention.

Every case is one call of one operator, as a serving program makes it: buffers for the results are the
program's own and are written again by each call. ``run`` computes the plain form with elementary torch
operations in 32 bits, or, where ``own`` is true, calls the framework's operators.
"""
import math
import os
import sys

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}


# ------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # one new audio token per CFG arm over a 30 s cache: the smallest call, latency counts
        dict(name="attn_token", op="attn", type="bf16", B=2, Sq=1, Sk=704, H=8, Hk=8, d=64, layer=3, causal=True,
             lens="ragged", mask=False),
        # one token for each of four sequences over a long cache of shared kv heads: reads the cache once
        dict(name="attn_cache", op="attn", type="bf16", B=4, Sq=1, Sk=32768, H=32, Hk=8, d=64, layer=6, causal=True,
             lens="ragged", mask=False),
        # a joint block of the 8 s geometry (latent + clip + text rows, the text padding masked)
        dict(name="attn_joint_8s", op="attn", type="bf16", B=2, Sq=329, Sk=329, H=8, Hk=8, d=64, layer=1, causal=False,
             lens="full", mask=True),
        # a joint block of the 30 s geometry with 32-wide maps
        dict(name="attn_joint_30s", op="attn", type="f16", B=2, Sq=1021, Sk=1021, H=16, Hk=16, d=32, layer=9,
             causal=False, lens="full", mask=False),
        # a chunk of tokens appended to a cache of grouped kv heads, causal from the end
        dict(name="attn_chunk", op="attn", type="bf16", B=1, Sq=1024, Sk=9216, H=32, Hk=8, d=64, layer=4, causal=True,
             lens="full", mask=False),
        # every token of a short video (13 frames of 25 x 25 patches) against every other
        dict(name="attn_video", op="attn", type="bf16", B=1, Sq=8125, Sk=8125, H=16, Hk=16, d=64, layer=12,
             causal=False, lens="full", mask=False),
        # the queries and keys of one token per sequence, far into a stream
        dict(name="rope_token", op="rope", type="bf16", B=8, T=1, Y=1, X=1, Hq=16, Hk=16, D=64, axes=3, rot=32,
             layout="half", norm=True, order="token", start=70000),
        # the clip frames of two arms (8 frames of 14 x 14 patches) in the framework's 32-bit activations
        dict(name="rope_frames", op="rope", type="f32", B=2, T=8, Y=14, X=14, Hq=16, Hk=16, D=64, axes=3, rot=32,
             layout="interleaved", norm=True, order="token", start=0),
        # a video of 52 frames of 25 x 25 patches, written head-major for the attention
        dict(name="rope_video", op="rope", type="bf16", B=1, T=52, Y=25, X=25, Hq=32, Hk=32, D=64, axes=3, rot=32,
             layout="interleaved", norm=True, order="head", start=0),
        # one token per arm with a 32-bit residual stream
        dict(name="norm_token", op="norm", type="f16", xtype="f32", B=2, T=1, C=1024, post="rms", pre="rms",
             gate="batch", tanh=False, mod="batch", scale="one"),
        # a joint block's rows of the 8 s geometry, modulated per arm
        dict(name="norm_8s", op="norm", type="bf16", xtype="f32", B=2, T=329, C=1024, post="rms", pre="layer",
             gate="batch", tanh=False, mod="batch", scale="vector"),
        # the rows of two videos with a modulation of each token
        dict(name="norm_video", op="norm", type="bf16", xtype="bf16", B=2, T=16250, C=2048, post="rms", pre="layer",
             gate="token", tanh=True, mod="token", scale="scalar"),
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, spread over their logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _draw_attn(rng):
    form = rng.choice(("token", "self", "chunk"))
    Sk = _log(rng, 1, 32768 if form == "token" else 8192)
    Sq = rng.choice((1, 1, 1, 2, 3, 4)) if form == "token" else Sk if form == "self" else _log(rng, 2, 1024)
    Hk = rng.choice((1, 2, 3, 4, 8, 16))
    return dict(op="attn", type=rng.choice(("bf16", "f16")), B=_log(rng, 1, 8), Sq=Sq, Sk=Sk,
                H=Hk * rng.choice((1, 1, 2, 3, 4, 8)), Hk=Hk, d=rng.choice((32, 64)), layer=rng.randrange(0, 21),
                causal=form != "self" or rng.random() < 0.3, lens=rng.choice(("full", "ragged", "empty")),
                mask=rng.random() < 0.3)


def _draw_rope(rng):
    D = rng.choice((32, 64, 64, 96, 128))
    flat = rng.random() < 0.4
    return dict(op="rope", type=rng.choice(("bf16", "f16", "f32")), B=_log(rng, 1, 8), T=_log(rng, 1, 4096 if flat else 52),
                Y=1 if flat else _log(rng, 2, 25), X=1 if flat else _log(rng, 2, 25), Hq=rng.randrange(1, 33),
                Hk=rng.randrange(1, 33), D=D, axes=rng.choice((1, 2, 3)), rot=rng.choice((D // 2, D // 2, D // 4, D // 2 - 3)),
                layout=rng.choice(("interleaved", "half")), norm=rng.random() < 0.7, order=rng.choice(("token", "head")),
                start=rng.choice((0, 0, _log(rng, 1, 100000))))


def _draw_norm(rng):
    t, x = rng.choice((("bf16", "bf16"), ("f16", "f16"), ("f32", "f32"), ("bf16", "f32"), ("f16", "f32")))
    C = _log(rng, 64, 8192)
    return dict(op="norm", type=t, xtype=x, B=_log(rng, 1, 8), T=_log(rng, 1, 16250),
                C=C if rng.random() < 0.3 else max(64, C // 64 * 64), post=rng.choice(("none", "rms", "layer")),
                pre=rng.choice(("rms", "layer")), gate=rng.choice(("none", "batch", "token")), tanh=rng.random() < 0.5,
                mod=rng.choice(("none", "batch", "token")), scale=rng.choice(("one", "scalar", "vector")))


def draw(rng):
    make = rng.choice((_draw_attn, _draw_attn, _draw_rope, _draw_norm))
    most = [work(c) for c in listed()]
    flops = max(w["flops"] for w in most)
    nbytes = max(w["bytes"] for w in most)
    while True:
        c = make(rng)
        w = work(c)
        # the plain form holds both maps: no more (query, key) pairs than the largest listed case
        pairs = c["B"] * c["H"] * c["Sq"] * c["Sk"] if c["op"] == "attn" else 0
        if 0 < w["flops"] <= flops and w["bytes"] <= nbytes and pairs <= 16 * 8125 * 8125 and 3072 not in c.values():
            return c


# ------------------------------------------------------------------------- what a case's sizes mean
def _lens(c):
    """The keys that each sequence has: all, fewer from sequence to sequence, or none at all for the last."""
    n = [c["Sk"] - (b * c["Sk"]) // (2 * c["B"]) for b in range(c["B"])]
    if c["lens"] == "full":
        return [c["Sk"]] * c["B"]
    return n[:-1] + [0] if c["lens"] == "empty" else n


def _hidden(c, device):
    """[B, Sk], true where a key is masked: holes and a padded end, another one in each sequence."""
    j = torch.arange(c["Sk"], device=device)[None, :]
    b = torch.arange(c["B"], device=device)[:, None]
    return ((j + 3 * b) % 8 == 5) | ((j >= c["Sk"] - c["Sk"] // 6) & (b % 2 == 1))


def _pairs(c):
    """Visible (query, key) pairs of one head over the batch."""
    total = 0
    shown = ~_hidden(c, "cpu").numpy() if c["mask"] else np.ones((c["B"], c["Sk"]), bool)
    for b, n in enumerate(_lens(c)):
        seen = np.concatenate([[0], np.cumsum(shown[b, :n])])
        if c["causal"]:
            last = np.clip(np.arange(c["Sq"]) + n - c["Sq"] + 1, 0, n)
            total += int(seen[last].sum())
        else:
            total += int(seen[n]) * c["Sq"]
    return total


def work(c):
    if c["op"] == "attn":
        d2, e = 2 * c["d"], SIZE[c["type"]]
        keys = sum(_lens(c)) * c["Hk"] * 2 * d2 * e
        return {"bytes": float(keys + 2 * c["B"] * c["Sq"] * c["H"] * d2 * e + (c["B"] * c["Sk"] if c["mask"] else 0)),
                "flops": float(_pairs(c) * c["H"] * 12 * c["d"])}
    if c["op"] == "rope":
        S, e = c["T"] * c["Y"] * c["X"], SIZE[c["type"]]
        values = c["B"] * S * (c["Hq"] + c["Hk"]) * c["D"]
        return {"bytes": float(2 * values * e + S * c["axes"] * 4), "flops": float(values * (7 if c["norm"] else 3))}
    rows, e, x = c["B"] * c["T"], SIZE[c["type"]], SIZE[c["xtype"]]
    per = {"none": 0, "batch": c["B"], "token": rows}
    mod = (per[c["gate"]] + 2 * per[c["mod"]]) * c["C"] * e
    return {"bytes": float(rows * c["C"] * 2 * (x + e) + mod), "flops": float(rows * c["C"] * 16)}


# ------------------------------------------------------------------------------------------- inputs
def _framework():
    here = os.path.join(os.getcwd(), "thinksound-native_b200")
    if here not in sys.path:
        sys.path.insert(0, here)
    import tsn
    return tsn


_device = []


def _dev(tsn):
    """The program's one device handle, on torch's stream."""
    if not _device:
        _device.append(tsn.Device(0, stream=torch.cuda.current_stream().cuda_stream))
    return _device[0]


def _lambda_init(c):
    return 0.8 - 0.6 * math.exp(-0.3 * c["layer"])


def _prepare_attn(c, normal):
    t, d = DTYPES[c["type"]], c["d"]
    s = {"case": c, "lambda_init": _lambda_init(c), "eps": 1e-5}
    # queries and keys as a per-head RMSNorm with a gain of 1.2 leaves them
    s["q"] = (normal(c["B"], c["Sq"], c["H"], 2 * d) * 1.2).to(t)
    s["k"] = (normal(c["B"], c["Sk"], c["Hk"], 2 * d) * 1.2).to(t)
    s["v"] = normal(c["B"], c["Sk"], c["Hk"], 2 * d).to(t)
    s["vectors"] = [normal(d) * 0.1 for _ in range(4)]
    s["weight"] = 1.0 + 0.1 * normal(2 * d)
    s["out"] = torch.empty_like(s["q"])
    s["len"] = s["hidden"] = s["shown"] = None
    if c["lens"] != "full":
        s["len"] = torch.tensor(_lens(c), dtype=torch.int32, device="cuda")
        # what lies behind a sequence's end in its cache was never written
        dead = torch.arange(c["Sk"], device="cuda")[None, :] >= s["len"][:, None]
        s["k"].masked_fill_(dead[:, :, None, None], float("nan"))
        s["v"].masked_fill_(dead[:, :, None, None], float("nan"))
    if c["mask"]:
        s["shown"] = (~_hidden(c, "cuda")).to(torch.uint8)
    if own:
        tsn = _framework()
        s["op"] = tsn.DiffAttention(_dev(tsn), d, *s["vectors"], lambda_init=s["lambda_init"], norm_weight=s["weight"],
                                    eps=s["eps"])
    return s


def _axis_pairs(c):
    """Rotated pairs of each axis: time takes what height and width leave."""
    side = c["rot"] * 3 // 8 if c["axes"] == 3 else c["rot"] // 2
    return [c["rot"] - (c["axes"] - 1) * side] + [side] * (c["axes"] - 1)


def _frequencies(c):
    """[rot] turns per step of its axis, in 64 bits, and the axis of each pair."""
    turns, axis = [], []
    for a, n in enumerate(_axis_pairs(c)):
        turns += [10000.0 ** (-i / n) / (2 * math.pi) for i in range(n)]
        axis += [a] * n
    return np.array(turns), np.array(axis)


def _prepare_rope(c, normal):
    t, S = DTYPES[c["type"]], c["T"] * c["Y"] * c["X"]
    s = {"case": c, "eps": 1e-6}
    s["q"] = (normal(c["B"], S, c["Hq"], c["D"]) * 1.5).to(t)
    s["k"] = (normal(c["B"], S, c["Hk"], c["D"]) * 0.7).to(t)
    grid = torch.stack(torch.meshgrid(*(torch.arange(n, device="cuda") for n in (c["T"], c["Y"], c["X"])), indexing="ij"), -1)
    s["pos"] = (grid.reshape(S, 3) + torch.tensor([c["start"], 0, 0], device="cuda"))[:, : c["axes"]].to(torch.int32).contiguous()
    s["qw"], s["kw"] = (1.0 + 0.1 * normal(c["D"]), 1.0 + 0.1 * normal(c["D"])) if c["norm"] else (None, None)

    def result(like):
        if c["order"] == "token":
            return torch.empty_like(like)
        return torch.empty(like.transpose(1, 2).shape, dtype=t, device="cuda").transpose(1, 2)

    s["q_out"], s["k_out"] = result(s["q"]), result(s["k"])
    # the plain form's plan: turns per step as 64-bit fractions (products wrap at whole turns), and each pair's axis
    turns, axis = _frequencies(c)
    s["fraction"] = torch.from_numpy((turns * 2.0 ** 64).astype(np.uint64).view(np.int64)).cuda()
    s["axis"] = torch.from_numpy(axis).cuda()
    if own:
        tsn = _framework()
        s["op"] = tsn.RopeAxes(_dev(tsn), c["D"], _axis_pairs(c), theta=10000.0, layout=c["layout"], q_norm=s["qw"],
                               k_norm=s["kw"], eps=s["eps"])
    return s


def _prepare_norm(c, normal):
    t, B, T, C = DTYPES[c["type"]], c["B"], c["T"], c["C"]
    s = {"case": c, "eps": 1e-6}
    s["x"] = (normal(B, T, C) * 2.0).to(DTYPES[c["xtype"]])
    s["y"] = (normal(B, T, C) * 3.0 + 0.2).to(t)

    def rows(kind):
        return None if kind == "none" else (0.3 * normal(B, 1 if kind == "batch" else T, C)).to(t)

    s["gate"], s["shift"], s["mod"] = rows(c["gate"]), rows(c["mod"]), rows(c["mod"])
    s["post_w"] = 1.0 + 0.1 * normal(C) if c["post"] != "none" else None
    s["post_b"] = 0.1 * normal(C) if c["post"] == "layer" else None
    s["pre_w"] = 1.0 + 0.1 * normal(C)
    s["pre_b"] = 0.1 * normal(C) if c["pre"] == "layer" else None
    s["scale"] = {"one": 1.0, "scalar": 0.9, "vector": None}[c["scale"]]
    if s["scale"] is None:
        s["scale"] = 1.0 + 0.1 * normal(C)
    s["x_out"], s["h"] = torch.empty_like(s["x"]), torch.empty_like(s["y"])
    if own:
        tsn = _framework()
        s["op"] = tsn.BlockNorm(_dev(tsn), C, post=c["post"], pre=c["pre"], post_weight=s["post_w"], post_bias=s["post_b"],
                                pre_weight=s["pre_w"], pre_bias=s["pre_b"], post_eps=s["eps"], pre_eps=s["eps"],
                                residual_scale=s["scale"], gate_tanh=c["tanh"])
    return s


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    make = {"attn": _prepare_attn, "rope": _prepare_rope, "norm": _prepare_norm}[case["op"]]
    return make(case, lambda *shape: torch.randn(shape, generator=g, device="cuda"))


# ------------------------------------------------------------------------------ the operators, plain
def _visible(s):
    """[B, Sq, Sk], true where a query sees a key: inside its sequence, not masked, and not after it."""
    c = s["case"]
    j = torch.arange(c["Sk"], device="cuda")
    n = torch.full((c["B"],), c["Sk"], device="cuda") if s["len"] is None else s["len"].long()
    seen = (j[None, :] < n[:, None])
    if s["shown"] is not None:
        seen = seen & (s["shown"] != 0)
    seen = seen[:, None, :].expand(-1, c["Sq"], -1)
    if c["causal"]:
        i = torch.arange(c["Sq"], device="cuda")
        seen = seen & (j[None, None, :] <= i[None, :, None] + (n[:, None, None] - c["Sq"]))
    return seen


def _map(q, k, seen, scale):
    """softmax(scale q k') over the visible keys, all zero in a row that sees none; q [B, Hk, G, Sq, d], k [B, Hk, 1, Sk, d]."""
    a = (q @ k.transpose(-1, -2)).mul_(scale).masked_fill_(~seen, -math.inf)
    a = a.sub_(a.amax(-1, keepdim=True).clamp(min=-3e38)).exp_()
    return a.div_(a.sum(-1, keepdim=True).clamp(min=1e-38))


def _plain_attn(s):
    c, d = s["case"], s["case"]["d"]
    B, Sq, Sk, Hk, G = c["B"], c["Sq"], c["Sk"], c["Hk"], c["H"] // c["Hk"]
    seen = _visible(s)
    dead = ~seen.any(1)[:, :, None, None]
    q = s["q"].float().view(B, Sq, Hk, G, 2 * d).permute(0, 2, 3, 1, 4)
    k = s["k"].float().masked_fill(dead, 0.0).view(B, Sk, Hk, 1, 2 * d).permute(0, 2, 3, 1, 4)
    v = s["v"].float().masked_fill(dead, 0.0).view(B, Sk, Hk, 1, 2 * d).permute(0, 2, 3, 1, 4)
    lq1, lk1, lq2, lk2 = s["vectors"]
    lam = (lq1 * lk1).sum().exp() - (lq2 * lk2).sum().exp() + s["lambda_init"]
    seen = seen[:, None, None]
    a = _map(q[..., :d], k[..., :d], seen, d ** -0.5)
    a -= lam * _map(q[..., d:], k[..., d:], seen, d ** -0.5)
    o = a @ v
    o = o * (o.square().mean(-1, keepdim=True) + s["eps"]).rsqrt() * s["weight"] * (1.0 - s["lambda_init"])
    return o.permute(0, 3, 1, 2, 4).reshape(s["q"].shape).to(s["q"].dtype)


def _rms(x, w, eps):
    return x * (x.square().mean(-1, keepdim=True) + eps).rsqrt() * w


def _rotate(x, w, eps, cos, sin, c):
    n, x = c["rot"], x.float()
    if w is not None:
        x = _rms(x, w, eps)
    u, v = (x[..., 0 : 2 * n : 2], x[..., 1 : 2 * n : 2]) if c["layout"] == "interleaved" else (x[..., :n], x[..., n : 2 * n])
    a, b = u * cos - v * sin, u * sin + v * cos
    turned = torch.stack((a, b), -1).flatten(-2) if c["layout"] == "interleaved" else torch.cat((a, b), -1)
    return torch.cat((turned, x[..., 2 * n :]), -1)


def _plain_rope(s):
    c = s["case"]
    # an angle is a step count times a fraction of a turn: whole turns fall off a 64-bit product, 24 bits of the rest are kept
    part = (s["pos"].long()[:, s["axis"]] * s["fraction"]) >> 40
    angle = part.float() * (2.0 * math.pi / 2 ** 24)
    cos, sin = angle.cos()[None, :, None, :], angle.sin()[None, :, None, :]
    return (_rotate(s["q"], s["qw"], s["eps"], cos, sin, c).to(s["q"].dtype),
            _rotate(s["k"], s["kw"], s["eps"], cos, sin, c).to(s["k"].dtype))


def _norm(u, kind, w, b, eps):
    if kind == "none":
        return u
    if kind == "layer":
        u = u - u.mean(-1, keepdim=True)
    u = u * (u.square().mean(-1, keepdim=True) + eps).rsqrt() * w
    return u if b is None else u + b


def _plain_norm(s):
    c = s["case"]
    n = _norm(s["y"].float(), c["post"], s["post_w"], s["post_b"], s["eps"])
    if s["gate"] is not None:
        g = s["gate"].float()
        n = n * (g.tanh() if c["tanh"] else g)
    x = s["x"].float() * s["scale"] + n
    h = _norm(x, c["pre"], s["pre_w"], s["pre_b"], s["eps"])
    if s["mod"] is not None:
        h = h * (1.0 + s["mod"].float()) + s["shift"].float()
    return x.to(s["x"].dtype), h.to(s["y"].dtype)


def run(s):
    op = s["case"]["op"]
    if not own:
        return {"attn": _plain_attn, "rope": _plain_rope, "norm": _plain_norm}[op](s)
    if op == "attn":
        s["op"](s["q"], s["k"], s["v"], s["out"], key_len=s["len"], key_mask=s["shown"], causal=s["case"]["causal"])
        return s["out"]
    if op == "rope":
        s["op"](s["q"], s["k"], s["pos"], s["q_out"], s["k_out"])
        return s["q_out"], s["k_out"]
    s["op"](s["x"], s["y"], gate=s["gate"], shift=s["shift"], scale=s["mod"], x_out=s["x_out"], h=s["h"])
    return s["x_out"], s["h"]


# --------------------------------------------------------------------- the definitions in 64 bits
def _exact_attn(s):
    c, d = s["case"], s["case"]["d"]
    if c["B"] * c["H"] * c["Sq"] * c["Sk"] > 2 ** 31:
        return None
    q, k, v = (s[n].double() for n in ("q", "k", "v"))
    lq1, lk1, lq2, lk2 = (x.double() for x in s["vectors"])
    lam = float(torch.exp(lq1 @ lk1) - torch.exp(lq2 @ lk2)) + s["lambda_init"]
    out = torch.zeros_like(q)
    for b, n in enumerate(_lens(c)):
        cols = torch.arange(n, device="cuda")
        if c["mask"]:
            cols = cols[~_hidden(c, "cuda")[b, :n]]
        if not len(cols):
            continue
        for h in range(c["H"]):
            g = h // (c["H"] // c["Hk"])
            vv = v[b, cols, g]
            o = 0.0
            for part, weight in ((slice(0, d), 1.0), (slice(d, 2 * d), -lam)):
                z = q[b, :, h, part] @ k[b, cols, g, part].T / math.sqrt(d)
                if c["causal"]:
                    late = cols[None, :] > torch.arange(c["Sq"], device="cuda")[:, None] + (n - c["Sq"])
                    z[late] = -math.inf
                o = o + weight * (torch.softmax(z, -1).nan_to_num(0.0) @ vv)
            out[b, :, h] = o / torch.sqrt((o * o).mean(-1, keepdim=True) + s["eps"]) * s["weight"].double() * (1.0 - s["lambda_init"])
    return out


def _exact_rope(s):
    c = s["case"]
    turns, axis = _frequencies(c)
    pos = s["pos"].cpu().numpy().astype(np.float64)[:, axis]
    angle = torch.from_numpy(2.0 * math.pi * np.mod(pos * turns, 1.0)).cuda()
    turn = torch.polar(torch.ones_like(angle), angle)[None, :, None, :]
    outs = []
    for x, w in ((s["q"], s["qw"]), (s["k"], s["kw"])):
        x = x.double()
        if w is not None:
            x = x / torch.sqrt(torch.mean(x ** 2, -1, keepdim=True) + s["eps"]) * w.double()
        y, n = x.clone(), c["rot"]
        first, second = (slice(0, 2 * n, 2), slice(1, 2 * n, 2)) if c["layout"] == "interleaved" else (slice(0, n), slice(n, 2 * n))
        z = torch.complex(x[..., first].contiguous(), x[..., second].contiguous()) * turn
        y[..., first], y[..., second] = z.real, z.imag
        outs.append(y)
    return tuple(outs)


def _exact_norm(s):
    c = s["case"]
    wide = {n: None if s[n] is None or isinstance(s[n], float) else s[n].double()
            for n in ("x", "y", "gate", "shift", "mod", "post_w", "post_b", "pre_w", "pre_b", "scale")}

    def normed(u, kind, w, b):
        if kind == "none":
            return u
        if kind == "layer":
            var, mean = torch.var_mean(u, -1, correction=0, keepdim=True)
            u = (u - mean) / torch.sqrt(var + s["eps"])
        else:
            u = u / torch.sqrt((u * u).mean(-1, keepdim=True) + s["eps"])
        return w * u + (0.0 if b is None else b)

    n = normed(wide["y"], c["post"], wide["post_w"], wide["post_b"])
    if wide["gate"] is not None:
        n = (torch.tanh(wide["gate"]) if c["tanh"] else wide["gate"]) * n
    x = wide["x"] * (s["scale"] if wide["scale"] is None else wide["scale"]) + n
    h = normed(x, c["pre"], wide["pre_w"], wide["pre_b"])
    if wide["mod"] is not None:
        h = h + h * wide["mod"] + wide["shift"]
    return x, h


def exact(case, seed):
    s = prepare(case, seed)
    return {"attn": _exact_attn, "rope": _exact_rope, "norm": _exact_norm}[case["op"]](s)
