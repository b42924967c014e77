"""Sparse attention over picked pages (tsn.SparseAttention) against 64 bits: the picks exactly, the attention over them, and the
operators of the cache run together as a stream of tokens."""
import math

import pytest
import torch

import tsn
from paged_plain import Batch, attention, choose, within

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    d = tsn.Device(0, stream=torch.cuda.current_stream().cuda_stream)
    yield d
    d.close()


def check(dev, batch, H, picks, first=1, last=1, means=None, q=None, values=True):
    q = batch.rows(H) if q is None else q
    if means is None:
        means = batch.normal(batch.P, batch.Hk, batch.D).to(batch.dtype)
    out = torch.full_like(q, 3.0)
    chosen = torch.full((batch.N, batch.Hk, picks), 77, dtype=torch.int32, device="cuda")
    op = tsn.SparseAttention(dev, batch.D, picks, first=first, last=last)
    op(q, batch.k, batch.v, means, batch.table, batch.lens, out, chosen, q_start=batch.q_start)
    dev.commit()
    n = batch.starts[-1]
    want = choose(batch, q, means, picks, first, last)
    assert torch.equal(chosen[:n].cpu(), want[:n]) if values else best_but_for_rounding(batch, q, means, chosen.cpu(), want)
    assert bool((chosen[n:] == 77).all()) and bool((out[n:] == 3.0).all())
    if values:
        o, bound = attention(batch, q, pages=chosen)
        assert within(out[:n], o[:n], bound[:n])
    return chosen


def best_but_for_rounding(batch, q, means, chosen, want):
    """Whether the picks that differ from `want` have the same exact scores up to the rounding of 64-bit sums. Of G D products, each
    exact in 64 bits, any order of additions is off by at most (G D - 1) 2^-53 times the sum of their sizes, either score of a pair; the
    sums of numbers that do not fit 64 bits among them."""
    G = q.shape[1] // batch.Hk
    for row, b, p in batch.tokens():
        for h in range(batch.Hk):
            ours, theirs = set(chosen[row, h].tolist()), set(want[row, h].tolist())
            if len(ours) != len(theirs):
                return False
            x = q[row, h * G:(h + 1) * G].double().cpu()

            def score(page):
                terms = (x * means[batch.table[b, page].long(), h].double().cpu()).flatten().tolist()
                return math.fsum(terms), (len(terms) - 1) * 2.0 ** -53 * math.fsum(map(abs, terms))

            ours, theirs = sorted(map(score, ours - theirs)), sorted(map(score, theirs - ours))
            if any(abs(s - t) > 2 * max(e, f) for s, e in ours for t, f in theirs):
                return False
    return True


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "f16"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("page", [16, 64, 128])
@pytest.mark.parametrize("H,Hk", [(2, 2), (8, 2), (9, 1), (40, 2)])
def test_types_and_heads(dev, dtype, D, page, H, Hk):
    lens = [1, page, page + 1, 5 * page, 30 * page + 7]
    check(dev, Batch([1] * 5, lens, page=page, Hk=Hk, D=D, dtype=dtype, one=True), H, 6)


@pytest.mark.parametrize("picks,first,last", [(1, 0, 1), (2, 1, 1), (3, 0, 2), (4, 2, 2), (16, 0, 1), (33, 1, 4), (200, 1, 1), (1024, 3, 5)])
def test_picks(dev, picks, first, last):
    check(dev, Batch([1, 3, 0, 20], [900, 3, 50, 4000], page=16, extra=2, layout="head"), 4, picks, first, last)


@pytest.mark.parametrize("pages", [255, 256, 257, 511, 2049])
def test_numbers_of_pages(dev, pages):
    check(dev, Batch([2], [16 * pages - 3], Hk=1), 4, 17)


def test_ties_go_to_the_lowest_page(dev):
    """Means of a few whole numbers: most scores are shared by many pages, some are zero of either sign."""
    batch = Batch([1, 9], [5000, 3000], Hk=2, D=64)
    g = torch.Generator(device="cuda")
    g.manual_seed(1)
    means = torch.randint(-1, 2, (batch.P, 2, 64), generator=g, device="cuda").to(batch.dtype)
    means[::3] = 0.0
    means[::6] *= -1.0
    q = torch.randint(-1, 2, (batch.N, 4, 64), generator=g, device="cuda").to(batch.dtype)
    check(dev, batch, 4, 40, means=means, q=q)
    check(dev, batch, 4, 40, means=torch.zeros_like(means), q=q)


def test_scores_that_32_bits_do_not_tell_apart(dev):
    """A large part that all pages share, and differences below its 32-bit steps; numbers down to the subnormal ones."""
    for dtype in (torch.bfloat16, torch.float16):
        batch = Batch([4], [6000], Hk=1, D=128, dtype=dtype)
        means, q = torch.zeros(batch.P, 1, 128, device="cuda"), torch.zeros(batch.N, 2, 128, device="cuda")
        means[..., 0], q[..., 0] = 30000.0, 60000.0 if dtype is torch.float16 else 2.0 ** 30
        means[..., 1:] = batch.normal(batch.P, 1, 127) * 1e-3
        q[..., 1:] = batch.normal(batch.N, 2, 127) * 1e-3
        check(dev, batch, 2, 20, means=means.to(dtype), q=q.to(dtype), values=False)   # scores of 10^8 have no f32 softmax
        small = 1e-39 if dtype is torch.bfloat16 else 3e-7
        check(dev, batch, 2, 20, means=(batch.normal(batch.P, 1, 128) * small).to(dtype))


def test_pages_that_are_none(dev):
    """They may be chosen, with the score of zero means, and add no keys."""
    batch = Batch([2, 3], [900, 700], spare=0)
    batch.table[0, 5:20] = -1
    batch.table[1, 7] = batch.P
    batch.table[1, -1] = 2 ** 31 - 1
    check(dev, batch, 4, 12)
    batch.lens_ = [901 + 20, 2]   # behind the table's end, before the sequence's start
    batch.lens = torch.tensor(batch.lens_, dtype=torch.int32, device="cuda")
    check(dev, batch, 4, 12)


def test_more_tokens_and_long_caches(dev):
    check(dev, Batch([60, 1, 130], [3000, 9000, 130], page=32, Hk=2, D=128), 8, 9)
    check(dev, Batch([1, 1], [100000, 60001], page=64, Hk=2, D=128, one=True), 8, 32, 1, 2)
    check(dev, Batch([1], [16384 * 16], page=16, Hk=1, D=64, spare=0), 2, 64)


def test_all_pages_picked_is_dense(dev):
    batch = Batch([1, 40], [700, 500], D=128)
    q, M = batch.rows(4), batch.M
    out, dense = torch.empty_like(q), torch.empty_like(q)
    means, chosen = batch.normal(batch.P, 2, 128).to(batch.dtype), torch.empty(batch.N, 2, M, dtype=torch.int32, device="cuda")
    tsn.SparseAttention(dev, 128, M)(q, batch.k, batch.v, means, batch.table, batch.lens, out, chosen, q_start=batch.q_start)
    tsn.PagedAttention(dev, 128)(q, batch.k, batch.v, batch.table, batch.lens, dense, q_start=batch.q_start, most=40)
    dev.commit()
    want, bound = attention(batch, q)
    assert within(out, want, bound) and within(dense, want, bound)


def test_captured_and_replayed(dev):
    batch = Batch([1, 1], [30000, 25000], page=64, D=128, Hk=1, one=True)
    q, stream = batch.rows(4), torch.cuda.Stream()
    means = batch.normal(batch.P, 1, 128).to(batch.dtype)
    own = tsn.Device(0, stream=stream.cuda_stream)
    out, chosen = torch.empty_like(q), torch.empty(2, 1, 16, dtype=torch.int32, device="cuda")
    op, graph = tsn.SparseAttention(own, 128, 16), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        op(q, batch.k, batch.v, means, batch.table, batch.lens, out, chosen)
    for lens in ([30000, 25000], [29000, 5], [700, 1000]):
        batch.lens_ = lens
        batch.lens.copy_(torch.tensor(lens, dtype=torch.int32))
        q.copy_(batch.rows(4))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(chosen.cpu(), choose(batch, q, means, 16, 1, 1))
        assert within(out, *attention(batch, q, pages=chosen))
    del graph
    own.close()


@pytest.mark.parametrize("chunks", [[1] * 40, [40], [7, 1, 20, 12], [33, 7]])
def test_a_stream_of_tokens(dev, chunks):
    """Tokens of three streams appended and attended to, a few at a time: pages, means, dense and sparse results are those of the
    cache in 64 bits after each step."""
    page, Hk, H, D, total, picks = 16, 2, 6, 64, sum(chunks), 2
    start = [0, 21, 150]
    batch = Batch([total] * 3, [s + total for s in start], page=page, Hk=Hk, D=D, dtype=torch.float16)
    means = torch.full((batch.P, Hk, D), float("nan"), dtype=batch.dtype, device="cuda")
    full = tsn.CacheAppend(dev, D, (D // 2,), layout="half")
    dense, sparse = tsn.PagedAttention(dev, D), tsn.SparseAttention(dev, D, picks)
    # what each stream holds before: appended at once, its keys as they come
    kept = [(batch.normal(s, Hk, D).to(batch.dtype), batch.normal(s, Hk, D).to(batch.dtype)) for s in start]
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    batch.k.fill_(float("nan"))
    batch.v.fill_(float("nan"))
    full(None, torch.cat([k for k, _ in kept]), torch.cat([v for _, v in kept]), batch.k, batch.v, batch.table, ints(start),
         q_start=ints([0, 0, start[1], start[1] + start[2]]), means=means)
    at = list(start)
    for n in chunks:
        at = [a + n for a in at]
        step = Batch([n] * 3, at, page=page, Hk=Hk, D=D, dtype=batch.dtype, seed=n)
        step.table, step.P, step.M, step.k, step.v = batch.table, batch.P, batch.M, batch.k, batch.v
        q, k, v = step.rows(H), step.rows(Hk), step.rows(Hk, 1.0)
        out, out2 = torch.empty_like(q), torch.empty_like(q)
        chosen = torch.empty(3 * n, Hk, picks, dtype=torch.int32, device="cuda")
        full(q, k, v, batch.k, batch.v, batch.table, step.lens, q_start=step.q_start, means=means)
        dense(q, batch.k, batch.v, batch.table, step.lens, out, q_start=step.q_start, most=n)
        sparse(q, batch.k, batch.v, means, batch.table, step.lens, out2, chosen, q_start=step.q_start)
        dev.commit()
        assert within(out, *attention(step, q))
        assert torch.equal(chosen.cpu(), choose(step, q, means, picks, 1, 1))
        assert within(out2, *attention(step, q, pages=chosen))


@pytest.mark.parametrize("D,dtype", [(64, torch.float16), (128, torch.bfloat16)])
@pytest.mark.parametrize("last", [1, 3])
def test_many_tokens(dev, D, dtype, last):
    """Enough tokens that four share a block: of one sequence or of several, with rows of none behind."""
    counts = [301, 1, 2, 0, 250, 3, 40]
    lens = [n + 517 * b for b, n in enumerate(counts)]
    check(dev, Batch(counts, lens, page=16, Hk=2, D=D, dtype=dtype, extra=3, layout="head"), 6, 7, 1, last)


def test_many_single_tokens(dev):
    B = 330
    check(dev, Batch([1] * B, [1 + (97 * b) % 3000 for b in range(B)], page=32, Hk=4, D=128, one=True), 8, 6)
    batch = Batch([1] * B, [1 + (97 * b) % 700 for b in range(B)], page=16, Hk=4, D=64, one=True)
    g = torch.Generator(device="cuda")
    g.manual_seed(2)
    whole = lambda *s: torch.randint(-1, 2, s, generator=g, device="cuda").to(batch.dtype)  # noqa: E731
    check(dev, batch, 4, 9, means=whole(batch.P, 4, 64), q=whole(B, 4, 64))   # ties


def test_queries_and_means_that_are_not_finite(dev):
    """The picks are of the pages that there are, in order; attention with the other tokens is not touched."""
    batch = Batch([3, 2], [2000, 900], Hk=1, D=64)
    q, means = batch.rows(2), batch.normal(batch.P, 1, 64).to(batch.dtype)
    q[0, 0, 3], q[1, 1, 5], means[::7, 0, 9] = float("nan"), float("inf"), float("-inf")
    out, chosen = torch.full_like(q, 3.0), torch.full((5, 1, 12), 77, dtype=torch.int32, device="cuda")
    tsn.SparseAttention(dev, 64, 12)(q, batch.k, batch.v, means, batch.table, batch.lens, out, chosen, q_start=batch.q_start)
    dev.commit()
    for row, b, p in batch.tokens():
        c = chosen[row, 0].tolist()
        assert c == sorted(set(c)) and c[0] == 0 and c[-1] == p // 16
    want, bound = attention(batch, q, pages=chosen)
    assert within(out[2:], want[2:], bound[2:])
