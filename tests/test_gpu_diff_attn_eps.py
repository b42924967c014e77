"""Differential attention whose norm has eps 0: a row that sees no key is zero all the same, on every path (few rows in one
part and in several, tiles in one part and in several)."""
import pytest
import torch

import tsn
from test_gpu_diff_attn import formula, make, near, seen_of
from test_gpu_diff_attn import dev  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("typ,d", [("bf16", 64), ("f16", 32)])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("Sq,Sk", [(1, 17), (5, 300), (1, 20000), (60, 300), (64, 6000)])
def test_empty_rows_are_zero(dev, Sq, Sk, causal, typ, d):  # noqa: F811
    q, k, v, lams, w = make(Sq + Sk, typ, d, 4, Sq, Sk, 2, 2)
    lens = torch.tensor([Sk, 0, Sk, 3], dtype=torch.int32, device="cuda")
    mask = torch.ones(4, Sk, dtype=torch.uint8, device="cuda")
    mask[2] = 0
    seen = seen_of(4, Sq, Sk, lens, mask, causal)
    op = tsn.DiffAttention(dev, d, *lams, lambda_init=0.4, norm_weight=w, eps=0.0)
    out = torch.full_like(q, float("nan"))
    op(q, k, v, out, key_len=lens, key_mask=mask, causal=causal)
    dev.commit()
    empty = ~seen.any(-1)
    assert bool((out[empty] == 0).all())
    near(out, formula(q, k, v, lams, 0.4, w, 1e-300, seen), typ)   # the formula, 0 where it has 0 / 0
