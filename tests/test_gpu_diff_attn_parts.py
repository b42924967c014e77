"""Differential attention whose keys are split into parts (over the workspace for few rows, over a cluster for tiles), against the
definition in 64 bits: sequences and masks that leave parts whole, cut, empty or wholly masked, and rows that see keys in some
parts only. Tolerances are those of test_gpu_diff_attn.py."""
import pytest
import torch

import tsn
from test_gpu_diff_attn import DT, check_case, make
from test_gpu_diff_attn import dev  # noqa: F401

pytestmark = pytest.mark.gpu
NAN, INF = float("nan"), float("inf")
SHAPES = [(1, 6000), (4, 2100), (9, 4097), (60, 6000), (300, 2048)]


@pytest.mark.parametrize("typ,d", [("bf16", 64), ("f16", 64), ("bf16", 32), ("f16", 32)])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("Sq,Sk", SHAPES)
def test_lengths_that_leave_parts_empty(dev, Sq, Sk, causal, typ, d):  # noqa: F811
    lens = torch.tensor([Sk, 0, 1, 64, Sk // 3, Sk - 1, Sq // 2], dtype=torch.int32, device="cuda")
    q, k, v, lams, w = make(Sq + Sk + d, typ, d, 7, Sq, Sk, 4, 2)
    dead = (torch.arange(Sk, device="cuda")[None] >= lens[:, None])[:, :, None, None]
    for fill in (NAN, -INF):
        k.masked_fill_(dead, fill)
        v.masked_fill_(dead, fill)
        check_case(dev, q, k, v, lams, w, typ, lens=lens, causal=causal)


@pytest.mark.parametrize("typ,d", [("bf16", 64), ("f16", 32)])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("Sq,Sk", SHAPES)
def test_masks_that_hide_parts(dev, Sq, Sk, causal, typ, d):  # noqa: F811
    q, k, v, lams, w = make(Sq * 3 + Sk, typ, d, 6, Sq, Sk, 4, 2)
    mask = torch.ones(6, Sk, dtype=torch.uint8, device="cuda")
    mask[0, :Sk // 2] = 0                    # the first parts
    mask[1, Sk // 4:] = 0                    # the last ones
    mask[2] = 0                              # all
    mask[3, ::5] = 0                         # holes in every part
    mask[4] = 0
    mask[4, Sk - 1] = 1                      # one key, in the last part
    mask[5, Sk // 3:Sk - Sk // 3] = 0        # the middle ones
    hidden = (mask == 0)[:, :, None, None]
    lens = torch.tensor([Sk, Sk, Sk, Sk - 7, Sk, Sk // 2], dtype=torch.int32, device="cuda")
    for fill in (NAN, INF, torch.finfo(DT[typ]).min):
        k.masked_fill_(hidden, fill)
        v.masked_fill_(hidden, fill)
        check_case(dev, q, k, v, lams, w, typ, mask=mask, causal=causal)
    check_case(dev, q, k, v, lams, w, typ, mask=mask, lens=lens, causal=causal)


@pytest.mark.parametrize("Sq,Sk", SHAPES)
def test_a_value_that_is_not_finite_in_one_part(dev, Sq, Sk):  # noqa: F811
    """It makes the rows that see it NaN, whichever part it lies in, and touches no other row."""
    q, k, v, lams, w = make(7 * Sq + Sk, "bf16", 64, 2, Sq, Sk, 2, 2)
    for causal in (False, True):
        clean = check_case(dev, q, k, v, lams, w, "bf16", causal=causal)
        op = tsn.DiffAttention(dev, 64, *lams, lambda_init=0.4, norm_weight=w, eps=1e-5)
        for at in (0, Sk // 2, Sk - Sq // 2 - 1):
            for fill in (NAN, INF):
                bad = v.clone()
                bad[1, at, 0, 5] = fill
                out = torch.empty_like(q)
                op(q, k, bad, out, causal=causal)
                dev.commit()
                first = max(0, at - (Sk - Sq)) if causal else 0   # the first row that sees it
                assert bool(torch.isnan(out[1, first:, 0]).all())
                assert torch.equal(out[1, :first, 0], clean[1, :first, 0])
                assert torch.equal(out[0], clean[0]) and torch.equal(out[1, :, 1], clean[1, :, 1])
