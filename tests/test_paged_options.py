"""Options of the paged cache's objects that their arguments cannot hold are refused, not taken for others: a scale of 0, which stands
for the default, and numbers beyond 32 bits."""
import pytest

import tsn
from test_paged_host import Host, tensors


def test_scale():
    for make in (lambda s: tsn.PagedAttention(Host, 64, scale=s), lambda s: tsn.SparseAttention(Host, 64, 4, scale=s)):
        assert make(None)._a.scale == 0.0 and make(0.5)._a.scale == 0.5
        for zero in (0.0, -0.0, 0):
            with pytest.raises(ValueError):
                make(zero)


@pytest.mark.parametrize("n", [-1, -2 ** 32, 2 ** 32, 2 ** 32 + 5])
def test_numbers(n):
    op = tsn.PagedAttention(Host, 64)
    op._call = lambda dev, args: 0
    for option in ("window", "most"):
        op(**tensors(), **{option: 7})
        assert getattr(op._a, option) == 7
        with pytest.raises(ValueError):
            op(**tensors(), **{option: n})
    for options in (dict(picks=n), dict(picks=8, first=n), dict(picks=8, last=n)):
        with pytest.raises(ValueError):
            tsn.SparseAttention(Host, 64, **options)
