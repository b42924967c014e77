"""Appending where rows of no sequence lie before and behind the sequences' rows (a batch that starts anywhere in a larger
buffer): every sequence's tokens are appended, also where all of them are within the rows that one block takes."""
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


@pytest.mark.parametrize("counts", [[1], [3], [6], [2, 1, 3], [1, 0, 1]])
@pytest.mark.parametrize("rows", [40, 1500, 3000, 5000])
def test_rows_of_none_on_both_sides(dev, counts, rows):
    total = sum(counts)
    for start in (1, 2, 5, 8 * 100 + 1 if rows > 1000 else 9, rows - total - 1):
        batch = Batch(counts, [n + 5 + 9 * b for b, n in enumerate(counts)], extra=rows - total)
        starts = (batch.q_start + start).contiguous()
        q, k, v = batch.rows(4), batch.rows(2), batch.rows(2)
        q_out, kp, vp = torch.full_like(q, 3.0), torch.full_like(batch.k, 7.0), torch.full_like(batch.v, 7.0)
        means = torch.full((batch.P, 2, 64), 7.0, dtype=batch.dtype, device="cuda")
        k_want, v_want, q_want = kp.clone(), vp.clone(), q_out.clone()
        for row, b, p in batch.tokens():
            id = batch.mapped(b, p)
            k_want[id, p % 16], v_want[id, p % 16], q_want[start + row] = k[start + row], v[start + row], q[start + row]
        tsn.CacheAppend(dev, 64, (0,))(q, k, v, kp, vp, batch.table, batch.lens, q_out=q_out, q_start=starts, means=means)
        dev.commit()
        assert torch.equal(kp, k_want) and torch.equal(vp, v_want) and torch.equal(q_out, q_want), start
        touched = {batch.mapped(b, p) for row, b, p in batch.tokens()}
        assert all((id in touched) == bool((means[id] != 7.0).any()) for id in range(batch.P))
