"""Scores far beyond what an exponential can tell apart: the greatest one, or those that share it, take the row. Scores are products of
powers of two and small whole numbers, exact in f32, that lie at least as far apart as they are large / 8, so that the result in 64
bits is the mean of the greatest ones' values; on both kernels."""
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


@pytest.mark.parametrize("dtype,exponents", [(torch.float16, [(6, 6), (10, 8), (10, 12), (11, 13), (12, 12), (13, 12), (14, 13)]),
                                             (torch.bfloat16, [(10, 8), (15, 13), (20, 17), (40, 30), (60, 58), (60, 62)])], ids=["f16", "bf16"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("n,S,Hk,G", [(1, 90, 1, 2), (3, 3000, 1, 2), (300, 700, 8, 4), (64, 5000, 8, 4)])
def test_the_greatest_take_the_row(dev, dtype, D, exponents, n, S, Hk, G):
    for eq, ek in exponents:
        for factor in (1.0, 1.125, 1.75, 3.0):
            batch = Batch([n], [S], page=64, Hk=Hk, D=D, dtype=dtype)
            g = torch.Generator(device="cuda")
            g.manual_seed(eq)
            j, q = torch.arange(S, device="cuda"), torch.zeros(n, Hk * G, D, device="cuda")
            k = torch.zeros(S, Hk, D, device="cuda")
            k[..., 0] = torch.randint(-7, 8, (S, Hk), generator=g, device="cuda") * 2.0 ** ek
            q[..., 0] = factor * 2.0 ** eq
            q[1::2, :, 0] *= -1.0   # rows whose neighbours are of another sign, or small
            q[2::4, :, 0] *= 2.0 ** -eq
            batch.k[batch.table[0].long()[j // 64], j % 64] = k.to(dtype)
            q, out = q.to(dtype), torch.full((n, Hk * G, D), 3.0, dtype=dtype, device="cuda")
            tsn.PagedAttention(dev, D, scale=0.125)(q, batch.k, batch.v, batch.table, batch.lens, out, q_start=batch.q_start, most=n)
            dev.commit()
            want, bound = attention(batch, q, scale=0.125)
            assert bool(((out.double() - want).abs() <= bound).all()), (eq, ek, factor)


@pytest.mark.parametrize("scale", [1e-30, 1.2e-38, 1e-39, 1e-45])
@pytest.mark.parametrize("n,S,Hk,G", [(1, 90, 1, 2), (300, 700, 8, 4)])
def test_scales_of_almost_nothing(dev, scale, n, S, Hk, G):
    """Down to subnormal ones: seen keys share the row evenly, and rows that see nothing of a tile take nothing of it."""
    for causal, window in ((False, 0), (True, 0), (True, 20)):
        batch = Batch([n], [S], page=64, Hk=Hk, D=64)
        q = batch.rows(Hk * G)
        out = torch.full_like(q, 3.0)
        tsn.PagedAttention(dev, 64, scale=scale)(q, batch.k, batch.v, batch.table, batch.lens, out, q_start=batch.q_start, causal=causal,
                                                 window=window, most=n)
        dev.commit()
        want, bound = attention(batch, q, causal, window, scale=scale)
        assert bool(((out.double() - want).abs() <= bound).all()), (causal, window)
