"""A negative stride between the sequences' tables is refused whatever their width (tables of one entry were read before their start)."""
import pytest

import tsn
from test_paged_host import append, cache, plan, refused, rows

A = 1 << 20


@pytest.mark.parametrize("M", [1, 2, 4])
def test_negative_strides(M):
    c = cache(M=M, table_sb=-4)
    assert "stride" in refused("tsn_paged_attn", tsn.PagedAttnArgs(c=c, H=4, causal=1, q=rows(), out=rows()))
    assert "stride" in refused("tsn_cache_append", append(c=c), plan())
    assert "stride" in refused("tsn_sparse_attn", tsn.SparseAttnArgs(c=c, H=4, picks=4, first=1, last=1, q=rows(), out=rows(), means=rows(2), chosen=A))


def test_strides_that_are_not_taken():
    for c in (cache(M=0, table_sb=-4), cache(B=1, table_sb=-4), cache(M=1, table_sb=0)):
        assert refused("tsn_paged_attn", tsn.PagedAttnArgs(c=c, H=4, causal=1, q=rows(), out=rows())) is None
