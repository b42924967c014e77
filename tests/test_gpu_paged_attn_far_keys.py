"""Many keys far below one: together they still have their share, on both kernels and in both types, wherever the one lies (a
long cache whose first token takes most of the weight).

Tolerance: that of attention in 64 bits, and for f16 what is below its normal numbers: half a step of 2^-24 a key, where the greatest
probability is 2^7 at least, so 2^-32 of its share a key."""
import math

import pytest
import torch

import tsn
from paged_plain import Batch, attention

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    d = tsn.Device(0, stream=torch.cuda.current_stream().cuda_stream)
    yield d
    d.close()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "f16"])
@pytest.mark.parametrize("n,S,Hk,G", [(1, 131072, 1, 8), (4, 20000, 2, 4), (64, 40000, 8, 4), (300, 3000, 8, 4)])
@pytest.mark.parametrize("nats", [4.0, 11.0, 14.0, 15.5, 16.0, 17.2, 19.0])
def test_their_share(dev, dtype, n, S, Hk, G, nats):
    for spread in (0.0, 1.0):
        for one in (0, S // 2 + 5, S - n):
            batch = Batch([n], [S], page=128, Hk=Hk, D=64, dtype=dtype)
            j = torch.arange(S, device="cuda")
            ids = batch.table[0].long()[j // 128]
            k, v = torch.zeros(S, Hk, 64, device="cuda"), torch.ones(S, Hk, 64, device="cuda")
            k[..., 1] = spread * batch.normal(S, Hk)
            k[one, :, 0], v[one] = nats, 0.0   # its value is zero: the result is the share of the others
            batch.k[ids, j % 128], batch.v[ids, j % 128] = k.to(dtype), v.to(dtype)
            q = torch.zeros(n, Hk * G, 64, device="cuda")
            q[..., :2] = 8.0
            q, out = q.to(dtype), torch.full((n, Hk * G, 64), 3.0, dtype=dtype, device="cuda")
            tsn.PagedAttention(dev, 64)(q, batch.k, batch.v, batch.table, batch.lens, out, q_start=batch.q_start, most=n)
            dev.commit()
            want, bound = attention(batch, q)
            below = S * 2.0 ** -32 if dtype is torch.float16 else 0.0
            assert bool(((out.double() - want).abs() <= bound + below).all()), (spread, one, float(((out.double() - want).abs() / want.abs()).max()))
            if spread == 0.0 and one == 0:   # by the formula itself
                share = (S - n) * math.exp(-float(k[0, 0, 0].to(dtype)))   # the first of the new tokens sees S - n others
                assert abs(float(want[0, 0, 0]) * (1 + share) / share - 1.0) < 1e-6


@pytest.mark.parametrize("dtype,D", [(torch.float16, 64), (torch.float16, 128), (torch.bfloat16, 128)], ids=["f16-64", "f16-128", "bf16-128"])
@pytest.mark.parametrize("n,S,Hk,G", [(1, 900, 1, 2), (4, 9000, 1, 2), (140, 900, 4, 4), (64, 9000, 8, 4)])
def test_scores_that_rise_and_fall(dev, dtype, D, n, S, Hk, G):
    """The reference moves again and again, or the first keys hold it, over tens to thousands of log2 units."""
    for slope in (0.002, -0.002, 0.05, -0.05, 0.4):
        batch = Batch([n], [S], page=16, D=D, Hk=Hk, dtype=dtype)
        j = torch.arange(S, device="cuda")
        k = 0.3 * batch.normal(S, Hk, D)
        k[..., 0] = (slope * j)[:, None]
        batch.k[batch.table[0].long()[j // 16], j % 16] = k.to(dtype)
        q = batch.rows(Hk * G, 0.3)
        q[..., 0] = D ** 0.5
        out = torch.full_like(q, 3.0)
        tsn.PagedAttention(dev, D)(q, batch.k, batch.v, batch.table, batch.lens, out, q_start=batch.q_start, most=n)
        dev.commit()
        want, bound = attention(batch, q)
        # f32 scores: 2^-24 of their size (D + 1 products' sum and the factor) in the exponent, of either the key's or the greatest one's
        size = float(k[..., 0].abs().max()) + 4.0
        wide = 4 * size * 2.0 ** -23
        below = S * 2.0 ** -32 if dtype is torch.float16 else 0.0
        A = attention_sizes(batch, q)
        assert bool(((out.double() - want).abs() <= bound + wide * A + below * 6.0).all()), slope


def attention_sizes(batch, q):
    """sum w |v| of each element."""
    v = batch.v
    batch.v = v.abs()
    want, _ = attention(batch, q)
    batch.v = v
    return want
