"""Page picks of few tokens over many pages, where two or four blocks of a cluster share a token: every call's picks are the 64-bit
ones while other work holds some of the SMs, so that the blocks of a cluster come at different times."""
import pytest
import torch

import tsn
from paged_plain import Batch, choose

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("B,Hk,pages", [(1, 1, 1024), (1, 2, 2049), (3, 2, 1500), (1, 8, 4100), (9, 8, 1030)])
def test_beside_other_work(B, Hk, pages):
    stream, other = torch.cuda.Stream(), torch.cuda.Stream()
    dev = tsn.Device(0, stream=stream.cuda_stream)
    batch = Batch([1] * B, [16 * pages - 5 * b for b in range(B)], page=16, Hk=Hk, D=64, one=True, spare=0)
    means = batch.normal(batch.P, Hk, 64).to(batch.dtype)
    op = tsn.SparseAttention(dev, 64, 24)
    calls = []
    for _ in range(4):
        q = batch.rows(2 * Hk)
        calls.append((q, [torch.full((B, Hk, 24), 77, dtype=torch.int32, device="cuda") for _ in range(8)], choose(batch, q, means, 24, 1, 1)))
    a = torch.randn(1500, 1500, device="cuda")
    out, room = torch.empty_like(calls[0][0]), torch.empty_like(a)
    torch.cuda.synchronize()
    for r in range(8):
        with torch.cuda.stream(other):
            torch.mm(a, a, out=room)
        for q, chosen, _ in calls:
            op(q, batch.k, batch.v, means, batch.table, batch.lens, out, chosen[r])
    torch.cuda.synchronize()
    for _, chosen, want in calls:
        for c in chosen:
            assert torch.equal(c.cpu(), want)
    dev.close()
