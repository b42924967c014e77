"""Batches over a paged key/value cache for the tests, and what its operators give in 64 bits, token by token from the
formulas. Pages that a batch does not own, and slots behind a sequence's end, hold NaN."""
import math

import torch


class Batch:
    """`counts` new tokens and `lens` cached ones (the new included) of each sequence; `extra` rows behind the last sequence;
    `spare` entries of the tables behind each sequence's pages."""

    def __init__(self, counts, lens, page=16, Hk=2, D=64, dtype=torch.bfloat16, layout="token", extra=0, spare=1, one=False, seed=0,
                 device="cuda"):
        g = torch.Generator(device=device)
        g.manual_seed(seed)
        self.normal = lambda *s: torch.randn(s, generator=g, device=device)
        self.counts, self.lens_, self.page, self.Hk, self.D, self.dtype, self.device = counts, lens, page, Hk, D, dtype, device
        self.B, held = len(counts), [max(0, (n + page - 1) // page) for n in lens]
        self.P, self.M = sum(held) + 2, max(held + [0]) + spare
        order = torch.randperm(self.P, generator=g, device=device).to(torch.int32)
        self.table = torch.full((self.B, self.M), -1, dtype=torch.int32, device=device)
        at = 0
        for b, n in enumerate(held):
            self.table[b, :n] = order[at:at + n]
            at += n
        self.starts = [0]
        for n in counts:
            self.starts.append(self.starts[-1] + n)
        self.N = self.starts[-1] + extra
        ints = lambda x: torch.tensor(x, dtype=torch.int32, device=device)  # noqa: E731
        self.lens, self.q_start = ints(lens), None if one else ints(self.starts)
        self.k, self.v = (self.pages(layout) for _ in range(2))
        for b, n in enumerate(lens):
            for j in range(held[b]):
                m = min(page, n - j * page)
                for x, gain in ((self.k, 1.2), (self.v, 1.0)):
                    x[self.table[b, j].long(), :m] = (gain * self.normal(m, Hk, D)).to(dtype)

    def pages(self, layout, fill=float("nan")):
        P, page, Hk, D = self.P, self.page, self.Hk, self.D
        shape = {"token": (P, page, Hk, D), "head": (P, Hk, page, D), "page": (page, Hk, P, D)}[layout]
        t = torch.full(shape, fill, dtype=self.dtype, device=self.device)
        return {"token": lambda: t, "head": lambda: t.transpose(1, 2), "page": lambda: t.permute(2, 0, 1, 3)}[layout]()

    def rows(self, H, gain=1.2, dtype=None):
        return (gain * self.normal(self.N, H, self.D)).to(dtype or self.dtype)

    def tokens(self):
        """(row, sequence, place) of every new token."""
        for b in range(self.B):
            for i in range(self.counts[b]):
                yield self.starts[b] + i, b, self.lens_[b] - self.counts[b] + i

    def mapped(self, b, j):
        """The page of place j of sequence b, or None."""
        if not 0 <= j < self.M * self.page:
            return None
        id = int(self.table[b, j // self.page])
        return id if 0 <= id < self.P else None

    def cached(self, b):
        """Places of sequence b that lie in pages, and their keys and values in 64 bits."""
        n = max(0, min(self.lens_[b], self.M * self.page))
        j = torch.arange(n, device=self.device)
        ids = self.table[b].long()[j // self.page]
        j = j[(ids >= 0) & (ids < self.P)]
        ids = self.table[b].long()[j // self.page]
        return j, self.k[ids, j % self.page].double(), self.v[ids, j % self.page].double()


def attention(batch, q, causal=True, window=0, scale=None, pages=None):
    """(out, bound): the result in 64 bits, and what each element may be off by. pages[row][hk]: the pages that a token sees, or
    None for all. Rows of no sequence are NaN in both."""
    N, H, D = q.shape
    G, scale = H // batch.Hk, D ** -0.5 if scale is None else scale
    out = torch.full(q.shape, float("nan"), dtype=torch.float64, device=q.device)
    bound = out.clone()
    half = torch.finfo(q.dtype).eps / 2
    # probabilities and result are rounded to the type, half a step each: sum w_j half |v_j - o| <= half (A + |o|) with
    # A = sum w_j |v_j|, and half |o|. Scores, exponentials (2^-13 of each in bf16, 2^-18 in f16) and sums are f32: 2^-16 A covers
    # |s| 2^-22 for |s| up to 64.
    wide = 2.0 ** -12 if q.dtype is torch.bfloat16 else 2.0 ** -15
    for b in range(batch.B):
        if not batch.counts[b]:
            continue
        j, k, v = batch.cached(b)
        rows = slice(batch.starts[b], batch.starts[b + 1])
        p = torch.arange(batch.lens_[b] - batch.counts[b], batch.lens_[b], device=q.device)[:, None]
        seen = torch.ones(len(p), len(j), dtype=torch.bool, device=q.device)
        if causal:
            seen &= j[None] <= p
        if window:
            seen &= j[None] > p - window
        for h in range(batch.Hk):
            s = seen
            if pages is not None:
                listed = torch.zeros(len(p), batch.M + 1, dtype=torch.bool, device=q.device)
                chosen = pages[rows, h].long()
                listed.scatter_(1, torch.where(chosen < 0, batch.M, chosen), True)
                s = seen & listed[:, : batch.M][:, j // batch.page]
            s = s.repeat_interleave(G, 0)
            x = q[rows, h * G:(h + 1) * G].double().reshape(-1, D)
            a = (x @ k[:, h].T) * scale
            a = torch.where(s, a, torch.full_like(a, -math.inf))
            top = a.amax(-1, keepdim=True) if a.shape[1] else torch.zeros(len(a), 1, dtype=a.dtype, device=a.device)
            w = torch.where(s, torch.exp(a - torch.where(top == -math.inf, torch.zeros_like(top), top)), torch.zeros_like(a))
            w = w / w.sum(-1, keepdim=True).clamp(min=1e-300)
            # what is not seen has no effect whatever it holds; infinities and NaN that are seen enter as the arithmetic has it
            vh = v[:, h]
            clean = torch.where(vh.isfinite(), vh, torch.zeros_like(vh))
            o, A = w @ clean, w @ clean.abs()
            for x in (~vh.isfinite().all(-1)).nonzero().flatten().tolist():
                o += torch.where(s[:, x, None] & ~vh[x].isfinite(), vh[x], torch.zeros_like(vh[x]))
            out[rows, h * G:(h + 1) * G] = o.view(-1, G, D)
            bound[rows, h * G:(h + 1) * G] = (half * (A + 2 * o.abs()) + wide * A).view(-1, G, D)
    return out, bound


def within(got, want, bound):
    """Whether got is as far from want as bound says, and the same where want is not finite."""
    got, fine = got.double(), want.isfinite()
    return bool(((got - want).abs() <= bound)[fine].all()) and bool(((got == want) | (got.isnan() & want.isnan()))[~fine].all())


def choose(batch, q, means, picks, first, last):
    """The chosen pages [N, Hk, picks], int32 (0 in rows of no sequence)."""
    N, H, D = q.shape
    G = H // batch.Hk
    out = torch.zeros(N, batch.Hk, picks, dtype=torch.int32)
    qs = q.double().view(N, batch.Hk, G, D).sum(2)
    for row, b, p in batch.tokens():
        n = p // batch.page + 1 if 0 <= p < batch.M * batch.page else 0
        ids = batch.table[b, :n].long()
        valid = (ids >= 0) & (ids < batch.P)
        m = means[ids.clamp(0, batch.P - 1)].double() * valid[:, None, None]
        score = torch.einsum("hd,xhd->hx", qs[row], m).cpu()
        for h in range(batch.Hk):
            order = sorted(range(n), key=lambda x: (not (x < first or x > n - 1 - last), -float(score[h, x]), x))
            chosen = sorted(order[:picks])
            out[row, h] = torch.tensor(chosen + [-1] * (picks - len(chosen)), dtype=torch.int32)
    return out


def rotate(x, w, eps, pos, pairs, layout, theta=10000.0):
    """Norm and rotary positions of [rows, heads, D] in 64 bits, pos [rows, axes]."""
    x = x.double()
    if w is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * w.double()
    P, y, j = sum(pairs), x.clone(), 0
    for axis, n in enumerate(pairs):
        for i in range(n):
            angle = pos[:, axis].double() * theta ** (-i / n)
            cos, sin = torch.cos(angle)[:, None], torch.sin(angle)[:, None]
            e0, e1 = (2 * j, 2 * j + 1) if layout == "interleaved" else (j, j + P)
            y[..., e0], y[..., e1] = x[..., e0] * cos - x[..., e1] * sin, x[..., e0] * sin + x[..., e1] * cos
            j += 1
    return y
