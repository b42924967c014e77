"""Attention over a paged cache divides by the sum of the probabilities that its product takes, so that their rounding to 16 bits
cancels where all values are alike: the mean of equal values is that value, whatever the scores are.

The result is v to the bit: values are powers of two, whose neighbours are 2^-8 of them away in bf16 and 2^-11 in f16, so that the last
rounding returns them where what is held in 32 bits is off by less than half of that. Over n keys the product adds n / 16 times, each
off by 2^-23 of the sum at most, and the divisor n / 4 times in 2^-24: 2^-13 for 6000 keys. A divisor of unrounded
probabilities is off by up to 2^-8 and 2^-11."""
import pytest
import torch

import tsn
from paged_plain import Batch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    d = tsn.Device(0, stream=torch.cuda.current_stream().cuda_stream)
    yield d
    d.close()


def alike(batch):
    """Values that are a power of two for each head and column, in every slot that a sequence holds."""
    v = 2.0 ** torch.arange(batch.Hk * batch.D, device="cuda").remainder(7).sub(3).view(batch.Hk, batch.D)
    v[:, ::3] *= -1.0
    for b, n in enumerate(batch.lens_):
        j = torch.arange(n, device="cuda")
        batch.v[batch.table[b].long()[j // batch.page], j % batch.page] = v.to(batch.dtype)
    return v.to(batch.dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "f16"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("n,S,Hk,G", [(1, 60, 2, 4), (1, 6000, 1, 2), (4, 700, 2, 2), (300, 300, 2, 2), (300, 1500, 8, 4), (64, 6000, 8, 4)])
@pytest.mark.parametrize("gain", [0.6, 2.5])
def test_values_that_are_alike(dev, dtype, D, n, S, Hk, G, gain):
    batch = Batch([n, n], [S, (S + n) // 2], page=32, Hk=Hk, D=D, dtype=dtype)
    v = alike(batch)
    q = batch.rows(Hk * G, gain)
    out = torch.full_like(q, 3.0)
    for causal in (True, False):
        tsn.PagedAttention(dev, D)(q, batch.k, batch.v, batch.table, batch.lens, out, q_start=batch.q_start, causal=causal, most=n)
        dev.commit()
        assert torch.equal(out, v.repeat_interleave(G, 0).expand_as(out))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "f16"])
@pytest.mark.parametrize("n", [1, 4, 200])
def test_scores_that_agree(dev, dtype, n):
    """One key's score above all others, which agree: their probabilities are all rounded alike."""
    for below in (0.003, 0.3, 1.0, 2.7, 5.1):
        batch = Batch([n], [1500], page=64, Hk=8, D=64, dtype=dtype)
        v = alike(batch)
        j = torch.arange(1500, device="cuda")
        k = torch.zeros(1500, 8, 64, device="cuda")
        k[0, :, 0] = below
        batch.k[batch.table[0].long()[j // 64], j % 64] = k.to(dtype)
        q = torch.zeros(n, 16, 64, device="cuda")
        q[..., 0] = 8.0
        q, out = q.to(dtype), torch.full((n, 16, 64), 3.0, dtype=dtype, device="cuda")
        tsn.PagedAttention(dev, 64)(q, batch.k, batch.v, batch.table, batch.lens, out, q_start=batch.q_start, most=n)
        dev.commit()
        assert torch.equal(out, v.repeat_interleave(2, 0).expand_as(out)), below
