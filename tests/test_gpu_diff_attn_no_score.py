"""Differential attention over keys whose scores are -infinity: such a key has no share in its map on any path, as a masked one, and a
map that has no other key is zero (not a mean of the values, and not different from path to path)."""
import pytest
import torch

import tsn
from test_gpu_diff_attn import formula, make, near
from test_gpu_diff_attn import dev  # noqa: F401

pytestmark = pytest.mark.gpu
INF = float("inf")
SHAPES = [(1, 60), (4, 700), (2, 9000), (130, 128), (100, 500), (64, 6000), (40, 70)]


def case(Sq, Sk, typ, d):
    q, k, v, lams, w = make(5 * Sq + Sk + d, typ, d, 2, Sq, Sk, 4, 2)
    q[..., 0], q[..., d] = 1.0, 1.0   # an element of -inf in a key's map makes its scores in that map -inf
    return q, k, v, lams, w


def run(dev, q, k, v, lams, w, d, causal=False):  # noqa: F811
    op = tsn.DiffAttention(dev, d, *lams, lambda_init=0.4, norm_weight=w, eps=1e-5)
    out = torch.full_like(q, float("nan"))
    op(q, k, v, out, causal=causal)
    dev.commit()
    return out


@pytest.mark.parametrize("typ,d", [("bf16", 64), ("f16", 64), ("bf16", 32), ("f16", 32)])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("Sq,Sk", SHAPES)
def test_no_key_with_a_score(dev, Sq, Sk, causal, typ, d):  # noqa: F811
    q, k, v, lams, w = case(Sq, Sk, typ, d)
    k[..., 0], k[..., d] = -INF, -INF
    assert bool((run(dev, q, k, v, lams, w, d, causal) == 0).all())


@pytest.mark.parametrize("typ,d", [("bf16", 64), ("f16", 32)])
@pytest.mark.parametrize("Sq,Sk", SHAPES)
def test_some_keys_with_a_score(dev, Sq, Sk, typ, d):  # noqa: F811
    """The first half of the keys, or all but the first, have none: the result is that of the others."""
    for gone in (slice(0, Sk // 2), slice(1, Sk)):
        q, k, v, lams, w = case(Sq, Sk, typ, d)
        seen = torch.ones(2, Sq, Sk, dtype=torch.bool, device="cuda")
        seen[:, :, gone] = False
        want = formula(q, k, v, lams, 0.4, w, 1e-5, seen)
        k[:, gone, :, 0], k[:, gone, :, d] = -INF, -INF
        near(run(dev, q, k, v, lams, w, d), want, typ)


@pytest.mark.parametrize("typ,d", [("bf16", 64), ("f16", 32)])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("Sq,Sk", SHAPES)
def test_scores_that_are_nan_or_infinite(dev, Sq, Sk, causal, typ, d):  # noqa: F811
    """They make the rows that see their key NaN, in either map, and touch no other row."""
    q, k, v, lams, w = case(Sq, Sk, typ, d)
    clean = run(dev, q, k, v, lams, w, d, causal)
    for fill in (INF, float("nan")):
        for element in (0, d):
            for at in range(0, Sk, max(1, Sk // 7)):
                bad = k.clone()
                bad[1, at, 0, element] = fill
                out = run(dev, q, bad, v, lams, w, d, causal)
                first = max(0, at - (Sk - Sq)) if causal else 0   # the first row that sees it
                assert bool(torch.isnan(out[1, first:, :2]).all()), (fill, element, at)
                assert torch.equal(out[1, :first, :2], clean[1, :first, :2])
                assert torch.equal(out[0], clean[0]) and torch.equal(out[1, :, 2:], clean[1, :, 2:])
