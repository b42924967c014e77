"""Appending to a paged cache (tsn.CacheAppend) against 64 bits: types, layouts, ragged batches, pages that are none, means, and
what a call must leave alone."""
import pytest
import torch

import tsn
from paged_plain import Batch, rotate

pytestmark = pytest.mark.gpu
EPS = 1e-6


@pytest.fixture(scope="module")
def dev():
    d = tsn.Device(0, stream=torch.cuda.current_stream().cuda_stream)
    yield d
    d.close()


def close(got, want, wide, dtype):
    """Half a step of the type, and f32 arithmetic on numbers up to `wide`: norm (sum, rsqrt, two products), angle (2^-23 turns) and
    rotation are below 16 steps of 2^-24 and 2 pi 2^-23."""
    half = torch.finfo(dtype).eps / 2
    tiny = torch.finfo(dtype).tiny * torch.finfo(dtype).eps
    return bool(((got.double() - want).abs() <= half * want.abs() + 2.0 ** -19 * wide + tiny).all())


def check(dev, batch, Hq, xtype, pairs, layout, norm=True, positions=None, in_place=False, means=False, strided=True, queries=True, page_layout="token"):
    D, Hk, dtype = batch.D, batch.Hk, batch.dtype
    heads = Hq + 2 * Hk
    qkv = (1.5 * batch.normal(batch.N, heads, D)).to(xtype)
    q, k, v = qkv[:, :Hq], qkv[:, Hq:Hq + Hk], qkv[:, Hq + Hk:]
    if not strided:
        q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
    qw, kw = (1 + 0.1 * batch.normal(D), 1 + 0.1 * batch.normal(D)) if norm else (None, None)
    op = tsn.CacheAppend(dev, D, pairs, layout=layout, q_norm=qw, k_norm=kw, eps=EPS)
    kp, vp = batch.pages(page_layout), batch.pages(page_layout)
    kp.copy_(batch.k)
    vp.copy_(batch.v)
    mean = (0.1 * batch.normal(batch.P, Hk, D)).to(dtype) if means else None
    k_want, v_want, written = kp.double(), vp.double(), torch.zeros(kp.shape[:2], dtype=torch.bool, device="cuda")
    mean_want = mean.double() if means else None
    mean_new = torch.zeros(batch.P, dtype=torch.bool, device="cuda")
    q_out = q if in_place else torch.full((batch.N, Hq, D), 7.0, dtype=dtype, device="cuda")
    q_want, mine = q_out.double().clone(), torch.zeros(batch.N, dtype=torch.bool, device="cuda")
    place = torch.zeros(batch.N, 1, dtype=torch.int64, device="cuda")
    for row, b, p in batch.tokens():
        place[row, 0] = p
        mine[row] = True
    pos = place if positions is None else positions
    turned_q, turned_k = rotate(q, qw, EPS, pos, pairs, layout), rotate(k, kw, EPS, pos, pairs, layout)
    q_want[mine] = turned_q[mine]
    for row, b, p in batch.tokens():
        id = batch.mapped(b, p)
        if id is not None:
            k_want[id, p % batch.page], v_want[id, p % batch.page] = turned_k[row], v[row].double()
            written[id, p % batch.page] = True
    op(q if queries else None, k, v, kp, vp, batch.table, batch.lens, q_out=None if in_place or not queries else q_out, q_start=batch.q_start,
       pos=positions, means=mean)
    dev.commit()
    wide = turned_q.abs().amax()
    if queries:
        assert close(q_out[mine], q_want[mine], wide, dtype)
        assert torch.equal(q_out[~mine].double(), q_want[~mine])
    assert close(kp[written], k_want[written], turned_k.abs().amax(), dtype) and close(vp[written], v_want[written], 0.0, dtype)
    same = lambda x, y: bool(((x.double() == y) | (x.isnan() & y.isnan())).all())  # noqa: E731
    assert same(kp[~written], k_want[~written]) and same(vp[~written], v_want[~written])
    if means:
        for b in range(batch.B):
            touched = {p // batch.page: p for row, c, p in batch.tokens() if c == b and batch.mapped(b, p) is not None}
            for x, p in touched.items():
                id = int(batch.table[b, x])
                keys = kp[id, : p % batch.page + 1].double()   # as they are stored
                mean_want[id], mean_new[id] = keys.mean(0), True
                # half a step of the type and a sum of 1024 f32 values at most, each off by 2^-24 of the sum so far
                bound = torch.finfo(dtype).eps / 2 * mean_want[id].abs() + 2.0 ** -18 * keys.abs().mean(0)
                assert bool(((mean[id].double() - mean_want[id]).abs() <= bound).all())
        assert torch.equal(mean[~mean_new].double(), mean_want[~mean_new])


TYPES = [(torch.bfloat16, torch.bfloat16), (torch.float16, torch.float16), (torch.float32, torch.bfloat16), (torch.float32, torch.float16)]


@pytest.mark.parametrize("xtype,dtype", TYPES, ids=["bf16", "f16", "f32-bf16", "f32-f16"])
@pytest.mark.parametrize("layout", ["interleaved", "half"])
@pytest.mark.parametrize("D,rot", [(64, 32), (128, 40), (96, 41), (256, 128), (8, 4), (24, 5), (64, 0)])
def test_types_and_heads(dev, xtype, dtype, layout, D, rot):
    check(dev, Batch([1, 7, 0, 20], [1, 40, 9, 53], D=D, Hk=3, dtype=dtype), 5, xtype, (rot,), layout, means=True)


@pytest.mark.parametrize("page", [16, 32, 128, 1024])
@pytest.mark.parametrize("page_layout", ["token", "head", "page"])
def test_pages(dev, page, page_layout):
    check(dev, Batch([page + 3, 2, page], [page + 3, 3 * page + 1, 2 * page], page=page, layout=page_layout), 4, torch.bfloat16, (32,), "half",
          means=True, page_layout=page_layout)


def test_one_token_each(dev):
    for B in (1, 3, 40, 257):
        check(dev, Batch([1] * B, [1 + (37 * b) % 90 for b in range(B)], one=True, D=128, Hk=8), 32, torch.bfloat16, (64,), "half", means=True)


def test_many_sequences(dev):
    """More sequences than a search step takes, some of them empty, and rows of none behind."""
    counts = [(5 * b) % 4 for b in range(1100)]
    check(dev, Batch(counts, [n + (7 * b) % 20 for b, n in enumerate(counts)], extra=5), 2, torch.bfloat16, (16,), "interleaved",
          means=True)


def test_long_prompts(dev):
    check(dev, Batch([1500, 0, 900], [1500, 0, 1000], page=64, Hk=2), 4, torch.bfloat16, (32,), "half", norm=False, means=True)


@pytest.mark.parametrize("axes", [2, 3, 4])
def test_positions_of_several_axes(dev, axes):
    batch = Batch([9, 30], [20, 30], extra=2)
    g = torch.Generator(device="cuda")
    g.manual_seed(3)
    pos = torch.randint(-5000, 100000, (batch.N, axes), generator=g, device="cuda", dtype=torch.int32)
    check(dev, batch, 4, torch.float32, (5,) * axes, "half", positions=pos)


def test_in_place_and_without_queries(dev):
    for strided in (True, False):
        check(dev, Batch([9, 3], [20, 3]), 4, torch.bfloat16, (32,), "half", in_place=True, strided=strided)
        check(dev, Batch([9, 3], [20, 3]), 4, torch.bfloat16, (32,), "half", queries=False, strided=strided)


def test_pages_that_are_none(dev):
    """Tokens whose table entry is no page, or whose place the table does not reach, are dropped."""
    batch = Batch([40, 40, 5], [60, 45, 3], extra=1, spare=0)
    batch.table[0, 2] = -1
    batch.table[1, 1] = batch.P
    batch.table[1, 2] = 2 ** 31 - 1
    batch.lens_ = [60, 45 + 30, 3]   # the last tokens lie behind the table's end, the third sequence's before its start
    batch.lens = torch.tensor(batch.lens_, dtype=torch.int32, device="cuda")
    check(dev, batch, 4, torch.bfloat16, (32,), "half", means=True)


def test_far_offsets(dev):
    """Pages more than 2^32 bytes apart."""
    page, Hk, D = 1024, 8, 128
    P = 2 ** 31 // (page * Hk * D) + 3
    kp = torch.zeros(P, page, Hk, D, dtype=torch.float16, device="cuda")
    vp = torch.zeros_like(kp)
    table = torch.tensor([[P - 1, 0]], dtype=torch.int32, device="cuda")
    lens = torch.tensor([1024], dtype=torch.int32, device="cuda")
    k, v = (torch.randn(1, Hk, D, device="cuda", dtype=torch.float16) for _ in range(2))
    tsn.CacheAppend(dev, D, (0,))(None, k, v, kp, vp, table, lens)
    dev.commit()
    assert torch.equal(kp[P - 1, 1023], k[0]) and torch.equal(vp[P - 1, 1023], v[0])
    assert int(kp.count_nonzero()) == int(k.count_nonzero()) and int(vp.count_nonzero()) == int(v.count_nonzero())


def test_nothing_to_do(dev):
    batch = Batch([0, 0], [5, 0])
    x = torch.zeros(0, 2, 64, dtype=torch.bfloat16, device="cuda")
    before = batch.k.clone()
    tsn.CacheAppend(dev, 64, (32,))(x, x, x, batch.k, batch.v, batch.table, batch.lens, q_start=batch.q_start)
    dev.commit()
    assert torch.equal(before.view(torch.int16), batch.k.view(torch.int16))


def test_captured_and_replayed(dev):
    """A captured call takes the lengths, tables and tokens that its buffers hold at each replay."""
    batch = Batch([1, 4, 2], [90, 90, 90], D=64, Hk=2, page=16)
    stream = torch.cuda.Stream()
    own = tsn.Device(0, stream=stream.cuda_stream)
    op = tsn.CacheAppend(own, 64, (32,), layout="half", eps=EPS)
    q, k, v = batch.rows(4), batch.rows(2), batch.rows(2)
    q_out, means = torch.empty_like(q), torch.zeros(batch.P, 2, 64, dtype=batch.dtype, device="cuda")
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        op(q, k, v, batch.k, batch.v, batch.table, batch.lens, q_out=q_out, q_start=batch.q_start, means=means)
    for lens in ([90, 88, 60], [1, 4, 2], [33, 17, 90]):
        batch.lens_ = lens
        batch.lens.copy_(torch.tensor(lens, dtype=torch.int32))
        for x in (q, k, v):
            x.copy_(batch.normal(*x.shape))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for row, b, p in batch.tokens():
            pos = torch.tensor([[p]], device="cuda")
            id = batch.mapped(b, p)
            for got, x in ((q_out[row], q[row]), (batch.k[id, p % 16], k[row])):
                assert close(got, rotate(x[None], None, EPS, pos, (32,), "half")[0], x.abs().amax().double(), batch.dtype)
            assert torch.equal(batch.v[id, p % 16], v[row])
    del graph
    own.close()
