"""A wait that gives up in paged attention: the call reports it, and calls after it, whose keys meet in the same workspace, are right.
The waits of one block only count as run out (a test hook), in each block in turn; the calls between have other queries, so that sums left
over from a call before would show."""
import pytest
import torch

import tsn
from paged_plain import Batch, attention, within

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("S,Hk,G,D", [([9000], 8, 4, 128), ([4000, 300, 7000], 3, 2, 64), ([20000], 1, 8, 128)])
def test_calls_after_one(S, Hk, G, D):
    dev = tsn.Device(0, stream=torch.cuda.current_stream().cuda_stream)
    batch = Batch([1] * len(S), S, page=64, Hk=Hk, D=D, one=True)
    qs = [batch.rows(Hk * G) for _ in range(2)]
    wants = [attention(batch, q) for q in qs]
    op, out = tsn.PagedAttention(dev, D), torch.empty_like(qs[0])
    call = lambda i: op(qs[i], batch.k, batch.v, batch.table, batch.lens, out)  # noqa: E731
    call(0)
    dev.commit()
    reported = 0
    for block in list(range(148)) + [1000]:
        try:
            dev.selftest_paged_timeout(op._a, block)
        except tsn.TsnError as e:
            assert e.code == 8 and "gave up" in str(e)
            reported += 1
        for i in (1, 0):
            call(i)
            dev.commit()
            assert within(out, *wants[i]), block
    assert reported >= 20
    dev.close()


def test_refusals():
    dev = tsn.Device(0)
    with pytest.raises(tsn.TsnError) as e:
        dev.selftest_paged_timeout(tsn.PagedAttnArgs(), 0)
    assert e.value.code == 1
    dev.close()
