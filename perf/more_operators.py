"""Cases that measure the operators of the paged key/value cache: appending to it, attention of new tokens over it,
and sparse attention over the pages that a cheap score picks.

Every case is one call of one operator, as a serving program makes it for one layer: the caches, tables and buffers for the
results are the program's own, and results are written again by each call. ``run`` computes the plain form with elementary torch
operations in 32 bits (page scores and angles in 64), or, where ``own`` is true, calls the framework's operators.
"""
import math
import os
import sys

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}


# ------------------------------------------------------------------------------------------- cases
# B sequences; T new tokens of a sequence at most, `tokens` how they vary over the sequences; S cached tokens of the longest
# sequence, the new ones included; pages of `page` tokens; `layout`: tokens or heads first within a page.
def listed():
    return [
        # one new token for each of four short streams: the smallest call, latency counts
        dict(name="append_token", op="append", type="bf16", ctype="bf16", B=4, T=1, tokens="even", S=700, page=16, layout="token",
             Hq=16, Hk=16, D=64, axes=1, rot=32, turn="half", norm=True, means=False),
        # a step of 256 streams with grouped heads, keeping the page means that sparse attention needs
        dict(name="append_step", op="append", type="bf16", ctype="bf16", B=256, T=1, tokens="even", S=4000, page=64, layout="head",
             Hq=32, Hk=8, D=128, axes=1, rot=64, turn="half", norm=True, means=True),
        # frames of two videos (time, height, width) from 32-bit activations into a 16-bit cache
        dict(name="append_frames", op="append", type="f32", ctype="f16", B=2, T=1568, tokens="even", S=6272, page=32, layout="token",
             Hq=16, Hk=16, D=64, axes=3, rot=32, turn="interleaved", norm=True, means=False),
        # long prompts of different lengths at once, part of each head turned, with page means
        dict(name="append_prompts", op="append", type="bf16", ctype="bf16", B=8, T=8192, tokens="ragged", S=16384, page=64,
             layout="token", Hq=32, Hk=8, D=128, axes=1, rot=32, turn="half", norm=False, means=True),
        # one token for each of two short streams, small pages: the smallest call
        dict(name="attn_token", op="attn", type="bf16", B=2, T=1, tokens="even", S=704, page=16, layout="token", H=16, Hk=16, D=64,
             causal=True, window=0),
        # one token for each of 16 long streams with grouped heads: reads the cache once
        dict(name="attn_cache", op="attn", type="bf16", B=16, T=1, tokens="even", S=32768, page=64, layout="head", H=32, Hk=8, D=128,
             causal=True, window=0),
        # a few drafted tokens to check for each of 24 streams
        dict(name="attn_draft", op="attn", type="f16", B=24, T=4, tokens="ragged", S=8191, page=32, layout="token", H=32, Hk=8, D=128,
             causal=True, window=0),
        # prompts in pieces beside single tokens in one batch, each token seeing the last 2000 before it
        dict(name="attn_mixed", op="attn", type="f16", B=8, T=517, tokens="mixed", S=5333, page=16, layout="token", H=24, Hk=8, D=64,
             causal=True, window=2000),
        # a long piece of a prompt over what is cached before it
        dict(name="attn_chunk", op="attn", type="bf16", B=1, T=4096, tokens="even", S=16384, page=128, layout="token", H=32, Hk=8,
             D=128, causal=True, window=0),
        # one token for one stream, a few pages of a short cache
        dict(name="sparse_token", op="sparse", type="bf16", B=1, T=1, tokens="even", S=9001, page=32, layout="token", H=16, Hk=4, D=64,
             picks=8, first=1, last=2),
        # one token for each of eight very long streams
        dict(name="sparse_cache", op="sparse", type="bf16", B=8, T=1, tokens="even", S=131072, page=64, layout="head", H=32, Hk=8,
             D=128, picks=32, first=1, last=2),
        # a piece of a prompt, each token with pages of its own
        dict(name="sparse_chunk", op="sparse", type="f16", B=2, T=200, tokens="ragged", S=40000, page=64, layout="token", H=32, Hk=4,
             D=128, picks=16, first=1, last=1),
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, spread over their logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _draw_batch(rng, longest, tokens):
    T = rng.choice((1, 1, _log(rng, 2, 8), _log(rng, 9, tokens)))
    return dict(B=_log(rng, 1, 64), T=T, tokens=rng.choice(("even", "ragged", "mixed", "empty")) if T > 1 else "even",
                S=max(T, _log(rng, 1, longest)), page=rng.choice((16, 32, 64, 128)), layout=rng.choice(("token", "head")))


def _draw_heads(rng, name):
    Hk = rng.choice((1, 2, 3, 4, 8, 16))
    return {name: Hk * rng.choice((1, 2, 3, 4, 8, 16) if Hk < 8 else (1, 2, 4)), "Hk": Hk}


def _draw_append(rng):
    D = rng.choice((64, 64, 96, 128, 128, 256))
    t, ct = rng.choice((("bf16", "bf16"), ("f16", "f16"), ("f32", "bf16"), ("f32", "f16")))
    return dict(op="append", type=t, ctype=ct, **_draw_batch(rng, 16384, 8192), **_draw_heads(rng, "Hq"), D=D, axes=rng.choice((1, 1, 2, 3)),
                rot=rng.choice((D // 2, D // 2, D // 4, D // 2 - 3)), turn=rng.choice(("interleaved", "half")), norm=rng.random() < 0.6,
                means=rng.random() < 0.5)


def _draw_attn(rng):
    causal = rng.random() < 0.85
    return dict(op="attn", type=rng.choice(("bf16", "f16")), **_draw_batch(rng, 32768, 4096), **_draw_heads(rng, "H"),
                D=rng.choice((64, 128)), causal=causal, window=_log(rng, 1, 8192) if causal and rng.random() < 0.3 else 0)


def _draw_sparse(rng):
    picks = _log(rng, 2, 64)
    return dict(op="sparse", type=rng.choice(("bf16", "f16")), **_draw_batch(rng, 131072, 256), **_draw_heads(rng, "H"),
                D=rng.choice((64, 128)), picks=picks, first=rng.choice((0, 1, 1)), last=rng.choice((1, 1, 2) if picks > 2 else (1,)))


def draw(rng):
    make = rng.choice((_draw_append, _draw_attn, _draw_attn, _draw_sparse))
    op = make.__name__[6:]
    most = [(work(c), c["B"] * c["S"] * c["Hk"] * c["D"]) for c in listed() if c["op"] == op]
    flops, nbytes = max(w["flops"] for w, _ in most), max(w["bytes"] for w, _ in most)
    cached = max(n for _, n in most)
    while True:
        c = make(rng)
        w = work(c)
        if 0 < w["flops"] <= flops and w["bytes"] <= nbytes and c["B"] * c["S"] * c["Hk"] * c["D"] <= cached:
            return c


# ------------------------------------------------------------------------- what a case's sizes mean
def _counts(c):
    """New tokens of each sequence."""
    B, T = c["B"], c["T"]
    if c["tokens"] == "even":
        return [T] * B
    if c["tokens"] == "mixed":
        return [T - (b * T) // (2 * B) if b % 2 == 0 else 1 for b in range(B)]
    n = [T - (b * T) // (B + 1) for b in range(B)]
    return n[:-1] + [0] if c["tokens"] == "empty" and B > 1 else n


def _lens(c):
    """Cached tokens of each sequence, the new ones included."""
    return [max(n, c["S"] - (b * c["S"]) // (2 * c["B"])) for b, n in enumerate(_counts(c))]


def _pages(c):
    return [(n + c["page"] - 1) // c["page"] for n in _lens(c)]


def _between(lo, hi):
    """Sum of the whole numbers lo .. hi."""
    return (lo + hi) * (hi - lo + 1) // 2 if hi >= lo else 0


def _pairs(c):
    """Visible (query, key) pairs of one head over the batch, and the keys that some query sees."""
    pairs = keys = 0
    for n, S in zip(_counts(c), _lens(c)):
        if n == 0:
            continue
        if not c["causal"]:
            pairs, keys = pairs + n * S, keys + S
            continue
        # query at position p sees p + 1 keys, or the last `window` of them
        w, p0 = c["window"] or S, S - n
        full = max(0, min(n, w - 1 - p0))     # queries that see fewer than w
        pairs += _between(p0 + 1, p0 + full) + (n - full) * w
        keys += S - max(0, p0 - w + 1)
    return pairs, keys


def work(c):
    if c["op"] == "append":
        tokens, e, ce = sum(_counts(c)), SIZE[c["type"]], SIZE[c["ctype"]]
        values = tokens * (c["Hq"] + 2 * c["Hk"]) * c["D"]
        nbytes = values * (e + ce) + (tokens * c["axes"] * 4 if c["axes"] > 1 else 0)
        flops = tokens * (c["Hq"] + c["Hk"]) * c["D"] * (7 if c["norm"] else 3)
        if c["means"]:   # the keys that were in the touched pages before, and the means
            for n, S in zip(_counts(c), _lens(c)):
                if n:
                    first = (S - n) // c["page"]
                    nbytes += ((S - n) % c["page"] + ((S - 1) // c["page"] - first + 1)) * c["Hk"] * c["D"] * ce
                    flops += (S - first * c["page"]) * c["Hk"] * c["D"]
        return {"bytes": float(nbytes), "flops": float(flops)}
    e, rows = SIZE[c["type"]], sum(_counts(c))
    if c["op"] == "attn":
        pairs, keys = _pairs(c)
        return {"bytes": float((keys * c["Hk"] + rows * c["H"]) * 2 * c["D"] * e), "flops": float(pairs * c["H"] * 4 * c["D"])}
    nbytes, flops = rows * c["H"] * 2 * c["D"] * e + rows * c["Hk"] * c["picks"] * 4, 0
    for n, S in zip(_counts(c), _lens(c)):
        nbytes += min(S, n * c["picks"] * c["page"]) * c["Hk"] * 2 * c["D"] * e + ((S + c["page"] - 1) // c["page"] * c["Hk"] * c["D"] * e if n else 0)
        for p in range(S - n, S):
            own_page = p // c["page"]
            flops += own_page * c["Hk"] * 2 * c["D"] + (min(own_page, c["picks"] - 1) * c["page"] + p % c["page"] + 1) * c["H"] * 4 * c["D"]
    return {"bytes": float(nbytes), "flops": float(flops)}


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


def _cache(c, make):
    """[pages, page, Hk, D] as the layout has it in memory; a few pages more than the sequences hold."""
    P, page, Hk, D = sum(_pages(c)) + 3, c["page"], c["Hk"], c["D"]
    return make(P, page, Hk, D) if c["layout"] == "token" else make(P, Hk, page, D).transpose(1, 2)


def _batch(c, g):
    """What the scheduler hands over: the page tables (the pages of a sequence lie anywhere), lengths, and where each
    sequence's new tokens start."""
    held, counts = _pages(c), _counts(c)
    order = torch.randperm(sum(held) + 3, generator=g, device="cuda").to(torch.int32)
    table = torch.full((c["B"], max(held) + 2), -1, dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(held):
        table[b, :n] = order[at:at + n]
        at += n
    starts = [0]
    for n in counts:
        starts.append(starts[-1] + n)
    return {"case": c, "table": table, "lens": torch.tensor(_lens(c), dtype=torch.int32, device="cuda"), "rows": starts,
            "q_start": None if c["T"] == 1 and c["tokens"] == "even" else torch.tensor(starts, dtype=torch.int32, device="cuda")}


def _axis_pairs(c):
    """Rotated pairs of each axis: time takes what height and width leave."""
    side = c["rot"] * 3 // 8 if c["axes"] == 3 else c["rot"] // 2
    return [c["rot"] - (c["axes"] - 1) * side] + [side] * (c["axes"] - 1)


def _prepare_append(c, g, normal):
    s = _batch(c, g)
    N, t, ct = s["rows"][-1], DTYPES[c["type"]], DTYPES[c["ctype"]]
    s["eps"] = 1e-6
    # q, k and v are columns of one product's result
    heads = c["Hq"] + 2 * c["Hk"]
    qkv = normal(N, heads, c["D"]).to(t)
    s["q"], s["k"], s["v"] = qkv[:, : c["Hq"]], qkv[:, c["Hq"] : c["Hq"] + c["Hk"]], qkv[:, c["Hq"] + c["Hk"] :]
    s["qw"], s["kw"] = (1.0 + 0.1 * normal(c["D"]), 1.0 + 0.1 * normal(c["D"])) if c["norm"] else (None, None)
    s["q_out"] = torch.empty(N, c["Hq"], c["D"], dtype=ct, device="cuda")
    # what was cached before, and what sequences that are gone left behind
    s["k_pages"], s["v_pages"] = (_cache(c, lambda *n: normal(*n).to(ct)) for _ in range(2))
    s["means"] = (0.1 * normal(s["k_pages"].shape[0], c["Hk"], c["D"])).to(ct) if c["means"] else None
    s["pos"] = None
    if c["axes"] > 1:   # frames of 14 x 14 patches
        p = torch.cat([torch.arange(S - n, S, device="cuda") for n, S in zip(_counts(c), _lens(c))])
        s["pos"] = torch.stack((p // 196, p // 14 % 14, p % 14), -1)[:, : c["axes"]].to(torch.int32).contiguous()
    if own:
        tsn = _framework()
        s["op"] = tsn.CacheAppend(_dev(tsn), c["D"], _axis_pairs(c), theta=10000.0, layout=c["turn"], q_norm=s["qw"], k_norm=s["kw"],
                                  eps=s["eps"])
    return s


def _prepare_cached(c, g, normal):
    s = _batch(c, g)
    t = DTYPES[c["type"]]
    # queries and keys as a per-head norm with a gain of 1.2 leaves them
    s["q"] = (normal(s["rows"][-1], c["H"], c["D"]) * 1.2).to(t)
    s["out"] = torch.empty_like(s["q"])
    s["k_pages"] = _cache(c, lambda *n: (normal(*n) * 1.2).to(t))
    s["v_pages"] = _cache(c, lambda *n: normal(*n).to(t))
    for b, S in enumerate(_lens(c)):   # what lies behind a sequence's end was never written
        if S % c["page"]:
            last = s["table"][b, S // c["page"]].long()
            s["k_pages"][last, S % c["page"]:] = float("nan")
            s["v_pages"][last, S % c["page"]:] = float("nan")
    return s


def _prepare_attn(c, g, normal):
    s = _prepare_cached(c, g, normal)
    if own:
        tsn = _framework()
        s["op"] = tsn.PagedAttention(_dev(tsn), c["D"])
    return s


def _prepare_sparse(c, g, normal):
    s = _prepare_cached(c, g, normal)
    # keys that point the same way within a page, more or less, so that pages differ in their scores
    P = s["k_pages"].shape[0]
    s["k_pages"] += (normal(P, 1, c["Hk"], c["D"]) * 0.5).to(s["k_pages"].dtype)
    s["means"] = s["k_pages"].float().nan_to_num(0.0).mean(1).to(s["k_pages"].dtype)
    s["chosen"] = torch.empty(s["rows"][-1], c["Hk"], c["picks"], dtype=torch.int32, device="cuda")
    if own:
        tsn = _framework()
        s["op"] = tsn.SparseAttention(_dev(tsn), c["D"], c["picks"], first=c["first"], last=c["last"])
    return s


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    make = {"append": _prepare_append, "attn": _prepare_attn, "sparse": _prepare_sparse}[case["op"]]
    return make(case, g, lambda *shape: torch.randn(shape, generator=g, device="cuda"))


# ------------------------------------------------------------------------------ the operators, plain
def _turned(x, w, eps, cos, sin, c):
    n, x = c["rot"], x.float()
    if w is not None:
        x = x * (x.square().mean(-1, keepdim=True) + eps).rsqrt() * w
    inter = c["turn"] == "interleaved"
    u, v = (x[..., 0 : 2 * n : 2], x[..., 1 : 2 * n : 2]) if inter else (x[..., :n], x[..., n : 2 * n])
    a, b = u * cos - v * sin, u * sin + v * cos
    turned = torch.stack((a, b), -1).flatten(-2) if inter else torch.cat((a, b), -1)
    return torch.cat((turned, x[..., 2 * n :]), -1)


def _new_positions(s):
    """The sequence and the place in it of every new token."""
    c, device = s["case"], "cuda"
    counts, lens = _counts(c), _lens(c)
    seq = torch.cat([torch.full((n,), b, device=device) for b, n in enumerate(counts)])
    return seq, torch.cat([torch.arange(S - n, S, device=device) for n, S in zip(counts, lens)])


def _plain_append(s):
    c = s["case"]
    seq, at = _new_positions(s)
    axes = (at[:, None] if s["pos"] is None else s["pos"]).double()
    turns = torch.cat([10000.0 ** (-torch.arange(n, device="cuda", dtype=torch.float64) / n) for n in _axis_pairs(c)])
    axis = torch.cat([torch.full((n,), a, device="cuda") for a, n in enumerate(_axis_pairs(c))])
    angle = axes[:, axis] * turns
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    ct = s["q_out"].dtype
    s["q_out"].copy_(_turned(s["q"], s["qw"], s["eps"], cos, sin, c).to(ct))
    page, slot = s["table"][seq, at // c["page"]].long(), at % c["page"]
    s["k_pages"][page, slot] = _turned(s["k"], s["kw"], s["eps"], cos, sin, c).to(ct)
    s["v_pages"][page, slot] = s["v"].to(ct)
    if s["means"] is None:
        return s["q_out"], s["k_pages"], s["v_pages"]
    for b, (n, S) in enumerate(zip(_counts(c), _lens(c))):
        if n:
            first, last = (S - n) // c["page"], (S - 1) // c["page"]
            ids = s["table"][b, first : last + 1].long()
            there = (torch.arange(first * c["page"], (last + 1) * c["page"], device="cuda") < S).view(-1, c["page"], 1, 1)
            keys = s["k_pages"][ids].float().masked_fill(~there, 0.0)
            s["means"][ids] = (keys.sum(1) / there.sum(1)).to(ct)
    return s["q_out"], s["k_pages"], s["v_pages"], s["means"]


def _plain_attn(s):
    c, out = s["case"], s["out"]
    Hk, G, D = c["Hk"], c["H"] // c["Hk"], c["D"]
    for b, (n, S) in enumerate(zip(_counts(c), _lens(c))):
        if n == 0:
            continue
        ids = s["table"][b, : (S + c["page"] - 1) // c["page"]].long()
        k, v = (x[ids].flatten(0, 1)[:S].float().permute(1, 0, 2)[:, None] for x in (s["k_pages"], s["v_pages"]))
        j = torch.arange(S, device="cuda")
        step = max(1, 2 ** 29 // (c["H"] * S))
        for i in range(0, n, step):
            m = min(step, n - i)
            r = s["rows"][b] + i
            q = s["q"][r : r + m].float().view(m, Hk, G, D).permute(1, 2, 0, 3)
            a = (q @ k.transpose(-1, -2)) * D ** -0.5
            if c["causal"]:
                p = torch.arange(S - n + i, S - n + i + m, device="cuda")[:, None]
                hidden = j[None] > p
                if c["window"]:
                    hidden |= j[None] <= p - c["window"]
                a.masked_fill_(hidden, -math.inf)
            a = (a - a.amax(-1, keepdim=True)).exp_()
            o = (a @ v) / a.sum(-1, keepdim=True)
            out[r : r + m] = o.permute(2, 0, 1, 3).reshape(m, c["H"], D).to(out.dtype)
    return out


def _plain_sparse(s):
    c, out, chosen = s["case"], s["out"], s["chosen"]
    Hk, G, D, K, page = c["Hk"], c["H"] // c["Hk"], c["D"], c["picks"], c["page"]
    for b, (n, S) in enumerate(zip(_counts(c), _lens(c))):
        M = (S + page - 1) // page
        ids = s["table"][b, :M].long()
        means = s["means"][ids].double().permute(1, 2, 0)                                  # [Hk, D, M]
        step = max(1, 2 ** 27 // (Hk * max(M, K * page * D)))
        for i in range(0, n, step):
            m = min(step, n - i)
            r = s["rows"][b] + i
            p = torch.arange(S - n + i, S - n + i + m, device="cuda")
            q = s["q"][r : r + m].view(m, Hk, G, D)
            score = (q.double().sum(2).transpose(0, 1) @ means).transpose(0, 1)             # [m, Hk, M]
            j, mine = torch.arange(M, device="cuda"), (p // page)[:, None]
            always = (j < c["first"]) | (j > mine - c["last"])
            score = score.masked_fill(always[:, None], math.inf).masked_fill((j > mine)[:, None], -math.inf)
            best = score.sort(dim=-1, descending=True, stable=True)[1][..., :K]
            best = torch.where(best > mine[:, None], M, best).sort(-1)[0]                   # in order, M: none
            if K > M:
                best = torch.cat((best, torch.full((m, Hk, K - M), M, device="cuda")), -1)
            chosen[r : r + m] = torch.where(best == M, -1, best).to(torch.int32)
            at = best.clamp(max=M - 1)
            heads = torch.arange(Hk, device="cuda")[None, :, None]
            k, v = (x.permute(2, 0, 1, 3)[heads, ids[at]].flatten(2, 3).float() for x in (s["k_pages"], s["v_pages"]))
            place = (best[..., None] * page + torch.arange(page, device="cuda")).flatten(2)   # [m, Hk, K page]
            seen = place <= p[:, None, None]
            a = (q.float() @ k.masked_fill(~seen[..., None], 0.0).transpose(-1, -2)) * D ** -0.5
            a.masked_fill_(~seen[:, :, None], -math.inf)
            a = (a - a.amax(-1, keepdim=True)).exp_()
            o = (a @ v.masked_fill(~seen[..., None], 0.0)) / a.sum(-1, keepdim=True)
            out[r : r + m] = o.reshape(m, c["H"], D).to(out.dtype)
    return out, chosen


def run(s):
    c = s["case"]
    if not own:
        return {"append": _plain_append, "attn": _plain_attn, "sparse": _plain_sparse}[c["op"]](s)
    if c["op"] == "append":
        s["op"](s["q"], s["k"], s["v"], s["k_pages"], s["v_pages"], s["table"], s["lens"], q_out=s["q_out"], q_start=s["q_start"],
                pos=s["pos"], means=s["means"])
        return (s["q_out"], s["k_pages"], s["v_pages"]) + (() if s["means"] is None else (s["means"],))
    if c["op"] == "attn":
        s["op"](s["q"], s["k_pages"], s["v_pages"], s["table"], s["lens"], s["out"], q_start=s["q_start"], causal=c["causal"],
                window=c["window"], most=c["T"])
        return s["out"]
    s["op"](s["q"], s["k_pages"], s["v_pages"], s["means"], s["table"], s["lens"], s["out"], s["chosen"], q_start=s["q_start"])
    return s["out"], s["chosen"]


# --------------------------------------------------------------------- the definitions in 64 bits
def _exact_append(s):
    c = s["case"]
    table, page = s["table"].cpu(), c["page"]
    turns, axis = [], []
    for a, n in enumerate(_axis_pairs(c)):
        turns += [10000.0 ** (-i / n) / (2 * math.pi) for i in range(n)]
        axis += [a] * n
    turns, q_out = torch.tensor(turns, dtype=torch.float64, device="cuda"), torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    k_pages, v_pages = s["k_pages"].double(), s["v_pages"].double()
    means = None if s["means"] is None else s["means"].double()

    def head(x, w, phase):
        x = x.double()
        if w is not None:
            x = x / torch.sqrt(torch.mean(x ** 2, -1, keepdim=True) + s["eps"]) * w.double()
        n = c["rot"]
        first, second = (slice(0, 2 * n, 2), slice(1, 2 * n, 2)) if c["turn"] == "interleaved" else (slice(0, n), slice(n, 2 * n))
        z = torch.complex(x[..., first].contiguous(), x[..., second].contiguous()) * torch.polar(torch.ones_like(phase), phase)[:, None]
        y = x.clone()
        y[..., first], y[..., second] = z.real, z.imag
        return y

    for b, (n, S) in enumerate(zip(_counts(c), _lens(c))):
        if not n:
            continue
        rows = slice(s["rows"][b], s["rows"][b] + n)
        p = torch.arange(S - n, S, device="cuda")
        where = p[:, None] if s["pos"] is None else s["pos"][rows]
        phase = 2 * math.pi * torch.remainder(where[:, axis].double() * turns, 1.0)
        q_out[rows] = head(s["q"][rows], s["qw"], phase)
        k, v = head(s["k"][rows], s["kw"], phase), s["v"][rows].double()
        for pg in range((S - n) // page, (S - 1) // page + 1):
            lo, hi = max(S - n, pg * page), min(S, (pg + 1) * page)
            spot = int(table[b, pg])
            k_pages[spot, lo - pg * page : hi - pg * page] = k[lo - (S - n) : hi - (S - n)]
            v_pages[spot, lo - pg * page : hi - pg * page] = v[lo - (S - n) : hi - (S - n)]
            if means is not None:
                means[spot] = k_pages[spot, : hi - pg * page].mean(0)
    return (q_out, k_pages, v_pages) + (() if means is None else (means,))


def _softmax_rows(q, k, v, seen):
    """softmax(q k' / sqrt(D)) v for [R, D] rows over [n, D] keys, `seen` [R, n] or None."""
    z = q @ k.T / math.sqrt(q.shape[-1])
    if seen is not None:
        z = torch.where(seen, z, torch.full_like(z, -math.inf))
    return torch.softmax(z, -1) @ v


def _exact_attn(s):
    c = s["case"]
    if work(c)["flops"] > 4e12:
        return None
    out, G = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda"), c["H"] // c["Hk"]
    for b, (n, S) in enumerate(zip(_counts(c), _lens(c))):
        if not n:
            continue
        j = torch.arange(S, device="cuda")
        ids = s["table"][b].long()[j // c["page"]]
        for h in range(c["Hk"]):
            k, v = s["k_pages"][ids, j % c["page"], h].double(), s["v_pages"][ids, j % c["page"], h].double()
            for i in range(0, n, 512):
                m = min(512, n - i)
                r = slice(s["rows"][b] + i, s["rows"][b] + i + m)
                seen = None
                if c["causal"]:
                    back = torch.arange(S - n + i, S - n + i + m, device="cuda")[:, None] - j[None]
                    seen = (back >= 0) & (back < (c["window"] or S + 1))
                    seen = seen.repeat_interleave(G, 0)
                q = s["q"][r, h * G : (h + 1) * G].double().reshape(m * G, -1)
                out[r, h * G : (h + 1) * G] = _softmax_rows(q, k, v, seen).view(m, G, -1)
    return out


def _exact_sparse(s):
    c = s["case"]
    tokens = s["rows"][-1]
    if tokens * c["Hk"] > 4096:
        return None
    G, page, K = c["H"] // c["Hk"], c["page"], c["picks"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    chosen = torch.full((tokens, c["Hk"], K), -1, dtype=torch.int32)
    for b, (n, S) in enumerate(zip(_counts(c), _lens(c))):
        ids = s["table"][b].long()
        means = s["means"][ids[: (S + page - 1) // page]].double()
        scores = torch.einsum("thgd,mhd->thm", s["q"][s["rows"][b] : s["rows"][b] + n].double().view(n, c["Hk"], G, -1), means).cpu()
        for i in range(n):
            p, r = S - n + i, s["rows"][b] + i
            mine = p // page
            forced = [x for x in range(mine + 1) if x < c["first"] or x > mine - c["last"]]
            for h in range(c["Hk"]):
                value = scores[i, h]
                free = torch.tensor([x for x in range(mine + 1) if x not in forced], dtype=torch.long)
                rank = torch.argsort(-value[free], stable=True)[: K - len(forced)] if len(forced) < K else free[:0]
                picked = sorted(forced + free[rank].tolist()) if len(forced) < K else sorted(forced)[:K]
                chosen[r, h, : len(picked)] = torch.tensor(picked, dtype=torch.int32)
                j = torch.cat([torch.arange(x * page, min(p + 1, (x + 1) * page)) for x in picked]).cuda()
                k, v = s["k_pages"][ids[j // page], j % page, h].double(), s["v_pages"][ids[j // page], j % page, h].double()
                out[r, h * G : (h + 1) * G] = _softmax_rows(s["q"][r, h * G : (h + 1) * G].double(), k, v, None)
    return out, chosen.cuda()


def exact(case, seed):
    s = prepare(case, seed)
    return {"append": _exact_append, "attn": _exact_attn, "sparse": _exact_sparse}[case["op"]](s)
