"""Attention over a paged cache (tsn.PagedAttention) against 64 bits: lengths, masks, pages that end inside a tile or are none, NaN
where nothing is seen, ragged batches, strides, streams and graphs."""
import pytest
import torch

import tsn
from paged_plain import Batch, attention, within

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    d = tsn.Device(0, stream=torch.cuda.current_stream().cuda_stream)
    yield d
    d.close()


def check(dev, batch, H, causal=True, window=0, scale=None, most=None, q=None):
    q = batch.rows(H) if q is None else q
    out = torch.full_like(q, 3.0)
    op = tsn.PagedAttention(dev, batch.D, scale=scale)
    op(q, batch.k, batch.v, batch.table, batch.lens, out, q_start=batch.q_start, causal=causal, window=window,
       most=max(batch.counts + [0]) if most is None else most)
    dev.commit()
    want, bound = attention(batch, q, causal, window, scale)
    n = batch.starts[-1]
    assert within(out[:n], want[:n], bound[:n])
    assert bool((out[n:] == 3.0).all())   # rows of no sequence
    return out


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "f16"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("page", [16, 64, 256])
@pytest.mark.parametrize("H,Hk", [(2, 2), (8, 2), (3, 1), (16, 1)])
def test_one_token_each(dev, dtype, D, page, H, Hk):
    lens = [1, 2, 15, 16, 17, 63, 64, 65, 127, 128, 129, 300, 1000]
    check(dev, Batch([1] * len(lens), lens, page=page, Hk=Hk, D=D, dtype=dtype, one=True), H)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "f16"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("layout,page", [("token", 16), ("head", 32), ("page", 64), ("token", 128), ("head", 1024)])
def test_chunks(dev, dtype, D, layout, page):
    check(dev, Batch([200, 1, 0, 77, 300], [200, 400, 30, 500, 301], page=page, Hk=2, D=D, dtype=dtype, layout=layout, extra=3), 6)


@pytest.mark.parametrize("causal,window", [(False, 0), (True, 1), (True, 7), (True, 64), (True, 130), (True, 2 ** 30)])
@pytest.mark.parametrize("counts,lens", [([1, 1, 1], [1, 100, 700]), ([3, 2, 4], [3, 100, 700]), ([150, 40, 290], [150, 333, 700])])
def test_masks(dev, causal, window, counts, lens):
    for D, page in ((64, 16), (128, 64)):
        check(dev, Batch(counts, lens, page=page, D=D, Hk=2), 4, causal, window)


@pytest.mark.parametrize("n", [1, 2, 7, 8, 9, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 256, 257, 383, 511, 513])
def test_every_number_of_rows(dev, n):
    check(dev, Batch([n, 1], [n + 5, 90], page=32, Hk=1, D=128), 1)
    check(dev, Batch([n], [n], page=16, Hk=2, D=64), 6)


@pytest.mark.parametrize("G", [1, 2, 5, 8, 9, 16, 24, 33, 128])
def test_groups(dev, G):
    check(dev, Batch([1, 1], [70, 300], Hk=1, D=64, one=True), G)
    check(dev, Batch([3, 0, 30], [70, 10, 300], Hk=2, D=128), 2 * G)


def test_most_decides_nothing_but_the_kernel(dev):
    for counts, lens in (([1, 3, 2], [500, 900, 30]), ([100, 1, 5], [500, 900, 30])):
        for most in (0, 1, 3, 1000, 2 ** 31):
            check(dev, Batch(counts, lens, Hk=2, D=128), 8, most=most)


@pytest.mark.parametrize("counts", [[1, 1], [4, 2], [130, 60]])
def test_rows_that_see_nothing(dev, counts):
    """No tokens in the cache, fewer than new ones, pages that are none, a table that is too short."""
    for causal in (True, False):
        batch = Batch(counts, [300, 200])
        batch.lens_ = [0, counts[1] // 2]
        batch.lens = torch.tensor([-5 if counts[0] == 1 else 0, counts[1] // 2], dtype=torch.int32, device="cuda")
        check(dev, batch, 4, causal)
        batch = Batch(counts, [300, 200], spare=0)
        batch.table[0] = -1
        batch.table[1, 2:9] = 2 ** 31 - 1
        batch.table[1, 10] = batch.P
        check(dev, batch, 4, causal)
        batch = Batch(counts, [300, 200], spare=0)
        batch.lens_ = [500, 1000]   # the table ends before
        batch.lens = torch.tensor(batch.lens_, dtype=torch.int32, device="cuda")
        check(dev, batch, 4, causal)
        check(dev, batch, 4, True, window=20)


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("n", [1, 4, 100, 300])
def test_what_is_not_seen_has_no_effect(dev, bad, n):
    """Values that are not finite: of a later token, before the window, of a seen key."""
    batch = Batch([n, n], [n + 40, n + 70], page=32, D=64)
    for b in range(2):
        late = batch.lens_[b] - 1
        batch.v[batch.table[b, late // 32].long(), late % 32, 0, 5] = bad
        batch.v[batch.table[b, 0].long(), 3, 1, 60] = bad
    check(dev, batch, 4)
    check(dev, batch, 4, window=30)
    check(dev, batch, 4, causal=False)
    # keys: a hidden one has no effect
    batch = Batch([n, n], [n + 40, n + 70], page=32, D=64)
    for b in range(2):
        late = batch.lens_[b] - 1
        batch.k[batch.table[b, late // 32].long(), late % 32, :, 5] = bad
    q = batch.rows(4)
    out = torch.full_like(q, 3.0)
    tsn.PagedAttention(dev, 64)(q, batch.k, batch.v, batch.table, batch.lens, out, q_start=batch.q_start, most=n)
    dev.commit()
    rows = torch.cat([torch.arange(batch.starts[b], batch.starts[b + 1] - 1, device="cuda") for b in range(2)])
    want, bound = attention(batch, q)
    assert within(out[rows], want[rows], bound[rows])


def test_large_scores_and_moving_maxima(dev):
    """Scores that grow along the keys (the reference moves again and again), fall, and span hundreds."""
    for n, D in ((1, 128), (4, 64), (140, 128), (300, 64)):
        for slope in (0.05, -0.05, 0.4):
            batch = Batch([n], [900], page=16, D=D, Hk=1)
            j = torch.arange(900, device="cuda")
            ids = batch.table[0].long()[j // 16]
            k = torch.zeros(900, 1, D, device="cuda")
            k[:, 0, 0] = slope * j
            k[:, 0, 1:] = 0.3 * batch.normal(900, D - 1)
            batch.k[ids, j % 16] = k.to(batch.dtype)
            q = batch.rows(2, 0.3)
            q[..., 0] = D ** 0.5
            check(dev, batch, 2, q=q)


def test_scale(dev):
    for n in (1, 200):
        check(dev, Batch([n], [n + 300]), 4, scale=0.03)
        check(dev, Batch([n], [n + 300]), 4, scale=0.5)


@pytest.mark.parametrize("B,S,Hk,G", [(1, 40000, 1, 1), (1, 40000, 1, 8), (2, 20000, 8, 4), (70, 3000, 4, 2), (300, 333, 8, 1)])
def test_long_and_many(dev, B, S, Hk, G):
    check(dev, Batch([1] * B, [S - (b * S) // (2 * B) for b in range(B)], page=64, Hk=Hk, D=128, one=True), Hk * G)


@pytest.mark.parametrize("n,S,Hk,G", [(40, 9000, 1, 1), (200, 9000, 1, 2), (17, 20000, 2, 8), (600, 5000, 2, 4)])
def test_chunks_over_long_caches(dev, n, S, Hk, G):
    check(dev, Batch([n, 1, n // 2], [S, S // 2, S // 3], page=64, Hk=Hk, D=128), Hk * G)
    check(dev, Batch([n], [S], page=128, Hk=Hk, D=64, dtype=torch.float16), Hk * G, window=S // 2)


def test_many_ragged_sequences(dev):
    """More sequences than a warp scans at once, empty ones among them."""
    for top in (3, 40):
        counts = [(5 * b) % top for b in range(150)]
        check(dev, Batch(counts, [n + (13 * b) % 100 for b, n in enumerate(counts)], Hk=1, D=64, extra=7), 4)


@pytest.mark.parametrize("n,G", [(1, 1), (3, 2), (3, 4)])
@pytest.mark.parametrize("B", [1, 5, 60, 300])
def test_short_caches(dev, B, n, G):
    """Fewer keys than a share of the work holds: in units of their own, by the dozen a CTA, beside long ones, empty ones between."""
    lens = [1 + (7 * b) % 40 for b in range(B)]
    counts = [min(n, lens[b]) if b % 9 != 4 else 0 for b in range(B)]
    check(dev, Batch(counts, lens, Hk=3, D=64), 3 * G)
    lens[B // 2], counts[B // 2] = 2500, n
    check(dev, Batch(counts, lens, Hk=3, D=64), 3 * G)
    batch = Batch([1] * B, lens, Hk=3, D=128, one=True)
    batch.lens_ = [0 if b % 3 == 1 else S for b, S in enumerate(lens)]
    batch.lens = torch.tensor(batch.lens_, dtype=torch.int32, device="cuda")
    check(dev, batch, 3 * G)


def test_strides(dev):
    """Queries as columns of a wider product, results of padded heads, tables and lengths of a larger buffer, pages of another order."""
    for counts, lens in (([1, 1], [100, 300]), ([90, 200], [100, 300])):
        batch = Batch(counts, lens, D=64, Hk=2, layout="page")
        wide = batch.normal(batch.N, 12, 64).to(batch.dtype)
        q, out = wide[:, 3:7], torch.full((batch.N, 4, 72), 3.0, dtype=batch.dtype, device="cuda")
        table = torch.full((2, batch.M + 5), -7, dtype=torch.int32, device="cuda")
        table[:, : batch.M] = batch.table
        tsn.PagedAttention(dev, 64)(q, batch.k, batch.v, table[:, : batch.M], batch.lens, out[..., :64], q_start=batch.q_start, most=max(counts))
        dev.commit()
        want, bound = attention(batch, q)
        assert within(out[..., :64], want, bound) and bool((out[..., 64:] == 3.0).all())


def test_far_offsets(dev):
    """Pages more than 2^32 bytes apart."""
    page, Hk, D = 1024, 8, 128
    P = 2 ** 31 // (page * Hk * D) + 3
    kp = torch.empty(P, page, Hk, D, dtype=torch.float16, device="cuda")
    vp = torch.empty_like(kp)
    for n in (1, 80):
        batch = Batch([n], [1500], page=page, Hk=Hk, D=D, dtype=torch.float16, spare=0)
        q = batch.rows(16)
        want, bound = attention(batch, q)
        table = torch.tensor([[P - 1, P - 3]], dtype=torch.int32, device="cuda")
        for x, y in ((kp, batch.k), (vp, batch.v)):
            x[table[0].long()] = y[batch.table[0].long()]
        out = torch.empty_like(q)
        tsn.PagedAttention(dev, D)(q, kp, vp, table, batch.lens, out, q_start=batch.q_start, most=n)
        dev.commit()
        assert within(out, want, bound)


def test_shared_pages_and_repeats(dev):
    """Sequences with the same first pages; the same call twice gives the same bits."""
    for n in (1, 64):
        batch = Batch([n] * 4, [700 + n] * 4, D=128, Hk=2)
        batch.table[1:, :40] = batch.table[0, :40]
        a = check(dev, batch, 8, q=batch.rows(8))
        q = batch.rows(8)
        a, b = check(dev, batch, 8, q=q), check(dev, batch, 8, q=q)
        assert torch.equal(a, b)


@pytest.mark.parametrize("n", [1, 100])
def test_captured_and_replayed(dev, n):
    """A captured call takes what its buffers hold at each replay, lengths and tables among it."""
    batch = Batch([n, n], [4000, 2500], page=64, D=128, Hk=1)
    q, stream = batch.rows(4), torch.cuda.Stream()
    own = tsn.Device(0, stream=stream.cuda_stream)
    out, op, graph = torch.empty_like(q), tsn.PagedAttention(own, 128), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        op(q, batch.k, batch.v, batch.table, batch.lens, out, q_start=batch.q_start, most=n)
    for lens in ([4000, 2500], [n, 2500], [333, 1000]):
        batch.lens_ = lens
        batch.lens.copy_(torch.tensor(lens, dtype=torch.int32))
        q.copy_(batch.rows(4))
        out.fill_(3.0)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        want, bound = attention(batch, q)
        assert within(out, want, bound)
    del graph
    own.close()


def test_two_streams(dev):
    """Split keys on two handles and two streams at once, many times."""
    batches = [Batch([1], [30000 - 9000 * i], page=64, D=128, Hk=2, seed=i) for i in range(2)]
    qs = [b.rows(8) for b in batches]
    wants = [attention(b, q) for b, q in zip(batches, qs)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    devs = [tsn.Device(0, stream=s.cuda_stream) for s in streams]
    ops = [tsn.PagedAttention(d, 128) for d in devs]
    outs = [[torch.empty_like(q) for _ in range(20)] for q in qs]
    torch.cuda.synchronize()
    for r in range(20):
        for i in range(2):
            b = batches[i]
            ops[i](qs[i], b.k, b.v, b.table, b.lens, outs[i][r], q_start=b.q_start, most=1)
    torch.cuda.synchronize()
    for i in range(2):
        for r in range(20):
            assert within(outs[i][r], *wants[i])
    for d in devs:
        d.close()


def test_graphs_side_by_side(dev):
    """Captured calls whose keys are split, replayed on two streams at once beside eager calls of this handle and of differential
    attention, which share its workspace."""
    batches = [Batch([1], [26000 - 7000 * i], page=64, D=128, Hk=1, seed=i) for i in range(3)]
    qs = [b.rows(8) for b in batches]
    wants = [attention(b, q) for b, q in zip(batches, qs)]
    outs = [torch.empty_like(q) for q in qs]
    op = tsn.PagedAttention(dev, 128)
    call = lambda i: op(qs[i], batches[i].k, batches[i].v, batches[i].table, batches[i].lens, outs[i], q_start=batches[i].q_start, most=1)  # noqa: E731
    lam = 0.1 * torch.ones(64, device="cuda")
    diff = tsn.DiffAttention(dev, 64, lam, lam, lam, lam, lambda_init=0.3)
    k = torch.randn(1, 20000, 2, 128, device="cuda").bfloat16()
    dq, dout = torch.randn(1, 1, 8, 128, device="cuda").bfloat16(), torch.empty(1, 1, 8, 128, dtype=torch.bfloat16, device="cuda")
    diff(dq, k, k, dout)
    dev.commit()
    dwant = dout.clone()
    graphs, streams = [], [torch.cuda.Stream() for _ in range(2)]
    for i in range(2):
        tsn.check(tsn.lib().tsn_device_set_stream(dev.h, streams[i].cuda_stream))
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[i], stream=streams[i]):
            call(i)
    tsn.check(tsn.lib().tsn_device_set_stream(dev.h, torch.cuda.current_stream().cuda_stream))
    for o in outs + [dout]:
        o.fill_(3.0)
    torch.cuda.synchronize()
    for _ in range(20):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                graphs[i].replay()
        call(2)
        diff(dq, k, k, dout)
    dev.commit()
    torch.cuda.synchronize()
    for i in range(3):
        assert within(outs[i], *wants[i])
    assert torch.equal(dout, dwant)


def test_captured_twice_and_first_calls(dev):
    """The first call of a handle may be a captured one; sequences without tokens and rows without a sequence stay as they are."""
    stream = torch.cuda.Stream()
    own = tsn.Device(0, stream=stream.cuda_stream)
    batch = Batch([0, 3, 0], [50, 9000, 0], page=32, D=64, Hk=1, extra=2)
    q = batch.rows(4)
    out, op, graph = torch.full_like(q, 3.0), tsn.PagedAttention(own, 64), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        op(q, batch.k, batch.v, batch.table, batch.lens, out, q_start=batch.q_start, most=3)
        op(q, batch.k, batch.v, batch.table, batch.lens, out, q_start=batch.q_start, most=3)
    graph.replay()
    torch.cuda.synchronize()
    want, bound = attention(batch, q)
    assert within(out[:3], want[:3], bound[:3]) and bool((out[3:] == 3.0).all())
    del graph
    own.close()


def test_starts_that_are_none(dev):
    """Starts that do not ascend, or lie outside the rows, touch nothing outside the results; the other sequences are right."""
    for n in (2, 60):
        batch = Batch([n, n, n], [300, 200, 100], page=16, D=64, Hk=2)
        q = batch.rows(4)
        want, bound = attention(batch, q)
        for starts in ([0, n, 2 * n, 2 ** 31 - 1], [-7, n, 2 * n, 3 * n + 1], [0, n, n - 1, n - 1]):
            ids = torch.tensor(starts, dtype=torch.int32, device="cuda")
            room = torch.full((3 * n + 8, 4, 64), 3.0, dtype=q.dtype, device="cuda")
            tsn.PagedAttention(dev, 64)(q, batch.k, batch.v, batch.table, batch.lens, room[4:-4], q_start=ids, most=n)
            dev.commit()
            assert bool((room[:4] == 3.0).all()) and bool((room[-4:] == 3.0).all())
            assert within(room[4:4 + n], want[:n], bound[:n])
