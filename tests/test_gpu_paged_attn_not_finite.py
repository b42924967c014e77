"""Scores that are not finite, of keys that rows do see: NaN and +infinity make the row NaN, wherever among the keys of a step they
lie, and touch no other row; a key whose score is -infinity has no share. On both kernels, whole and in parts."""
import pytest
import torch

import tsn
from paged_plain import Batch, attention, within

pytestmark = pytest.mark.gpu
INF = float("inf")
# new tokens, cached ones, kv heads, heads of a group: few rows (whole, in parts), some, many (one tile of keys, several, in parts)
SHAPES = [(1, 90, 2, 2), (3, 9000, 1, 2), (300, 700, 1, 2), (40, 100, 2, 4), (300, 700, 8, 4), (64, 9000, 8, 4)]


@pytest.fixture(scope="module")
def dev():
    d = tsn.Device(0, stream=torch.cuda.current_stream().cuda_stream)
    yield d
    d.close()


def run(dev, batch, q, n):
    out = torch.full_like(q, 3.0)
    tsn.PagedAttention(dev, batch.D)(q, batch.k, batch.v, batch.table, batch.lens, out, q_start=batch.q_start, most=n)
    dev.commit()
    return out


def case(n, S, Hk, G, dtype, D):
    batch = Batch([n], [S], page=64, Hk=Hk, D=D, dtype=dtype)
    q = batch.rows(Hk * G)
    q[..., 3] = 1.0   # a key's element 3 that is not finite makes its score so
    return batch, q


@pytest.mark.parametrize("dtype,D", [(torch.bfloat16, 64), (torch.float16, 64), (torch.bfloat16, 128), (torch.float16, 128)],
                         ids=["bf16-64", "f16-64", "bf16-128", "f16-128"])
@pytest.mark.parametrize("n,S,Hk,G", SHAPES)
@pytest.mark.parametrize("fill", [float("nan"), INF])
def test_scores_that_are_nan_or_infinite(dev, n, S, Hk, G, dtype, D, fill):
    batch, q = case(n, S, Hk, G, dtype, D)
    clean, key = run(dev, batch, q, n), batch.k.clone()
    for base in (0, S - 16 - n // 2):   # seen by all rows; by some where there are many
        for place in range(max(0, base), max(0, base) + 16):
            batch.k.copy_(key)
            batch.k[batch.table[0, place // 64].long(), place % 64, 0, 3] = fill
            out = run(dev, batch, q, n)
            first = max(0, place - (S - n))   # the first token that sees it
            assert bool(out[first:, :G].isnan().all()), place
            assert torch.equal(out[:first, :G], clean[:first, :G]) and torch.equal(out[:, G:], clean[:, G:])


@pytest.mark.parametrize("dtype,D", [(torch.bfloat16, 64), (torch.float16, 128)], ids=["bf16-64", "f16-128"])
@pytest.mark.parametrize("n,S,Hk,G", SHAPES)
def test_scores_of_minus_infinity(dev, n, S, Hk, G, dtype, D):
    """Of some keys, of all but one, of all."""
    for gone in (slice(0, S // 2), slice(5, 37), slice(1, S), slice(0, S)):
        batch, q = case(n, S, Hk, G, dtype, D)
        j = torch.arange(S, device="cuda")[gone]
        batch.k[batch.table[0].long()[j // 64], j % 64, :, 3] = -INF
        assert within(run(dev, batch, q, n), *attention(batch, q))


@pytest.mark.parametrize("fill", [float("nan"), INF])
def test_queries(dev, fill):
    """A query that is not finite: its own row alone, in every place of a tile of rows."""
    for n in (1, 5, 130):
        batch, q = case(n, 400, 1, 2, torch.bfloat16, 64)
        batch.k[..., 3] = batch.k[..., 3].abs() + 0.5   # so that no score is -infinity
        clean = run(dev, batch, q, n)
        for row in range(0, n, max(1, n // 9)):
            bad = q.clone()
            bad[row, 1, 3] = fill
            out = run(dev, batch, bad, n)
            assert bool(out[row, 1].isnan().all())
            out[row, 1] = clean[row, 1]
            assert torch.equal(out, clean)


def test_picked_pages(dev):
    batch, q = case(3, 700, 1, 2, torch.float16, 64)
    means, chosen = torch.zeros(batch.P, 1, 64, dtype=batch.dtype, device="cuda"), torch.empty(3, 1, 4, dtype=torch.int32, device="cuda")
    op, key = tsn.SparseAttention(dev, 64, 4), batch.k.clone()
    for place in range(640, 656):   # of the tokens' own page
        batch.k.copy_(key)
        batch.k[batch.table[0, 10].long(), place % 64, 0, 3] = INF
        out = torch.full_like(q, 3.0)
        op(q, batch.k, batch.v, means, batch.table, batch.lens, out, chosen, q_start=batch.q_start)
        dev.commit()
        assert bool(out.isnan().all())


@pytest.mark.parametrize("dtype,D", [(torch.bfloat16, 64), (torch.float16, 128)], ids=["bf16-64", "f16-128"])
@pytest.mark.parametrize("n,S,Hk,G", SHAPES)
@pytest.mark.parametrize("bad", [INF, -INF, float("nan")])
def test_rows_without_a_score_are_zero(dev, n, S, Hk, G, dtype, D, bad):
    """All seen scores are -infinity: whatever the values hold, on every path."""
    batch, q = case(n, S, Hk, G, dtype, D)
    j = torch.arange(S, device="cuda")
    batch.k[batch.table[0].long()[j // 64], j % 64, :, 3] = -INF
    for places in ([0], [S - n], [3, S // 2, S - 1]):
        v = batch.v.clone()
        for place in places:
            batch.v[batch.table[0, place // 64].long(), place % 64, :, 7] = bad
        assert bool((run(dev, batch, q, n) == 0).all())
        batch.v.copy_(v)


@pytest.mark.parametrize("dtype,D", [(torch.bfloat16, 64), (torch.float16, 64), (torch.float16, 128)], ids=["bf16-64", "f16-64", "f16-128"])
@pytest.mark.parametrize("n,S,Hk,G", SHAPES)
@pytest.mark.parametrize("bad", [INF, -INF, float("nan")])
def test_values_of_keys_without_weight(dev, n, S, Hk, G, dtype, D, bad):
    """A seen value that is not finite leaves its column so, however small its key's share is (it rounds to zero here), and touches
    neither the other columns nor the rows that do not see it."""
    batch, q = case(n, S, Hk, G, dtype, D)
    j = torch.arange(S, device="cuda")
    batch.k[batch.table[0].long()[j // 64], j % 64, :, 3] = 0.0
    for place in {1, S // 2, S - 1 - n // 2, S - 1}:
        k, v = batch.k.clone(), batch.v.clone()
        at = (batch.table[0, place // 64].long(), place % 64)
        batch.k[at][:, 3] = -2000.0   # 250 nats and 177 below the others
        clean, (_, bound) = run(dev, batch, q, n), attention(batch, q)
        batch.v[at][0, 7] = bad
        out = run(dev, batch, q, n)
        first = max(0, place - (S - n))
        assert not bool(out[first:, :G, 7].isfinite().any()), place
        out[first:, :G, 7] = clean[first:, :G, 7]
        batch.k.copy_(k)
        batch.v.copy_(v)
        assert torch.equal(out[:first], clean[:first])
        assert bool(((out.double() - clean.double()).abs() <= 2 * bound).all())   # either is within the bound of the exact one
