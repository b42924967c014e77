"""Differential attention: a map's divisor is the sum of the probabilities that its product with v takes, so their
rounding to 16 bits cancels where all values are alike, o = (1 - lambda) v whatever the scores are.

Tolerance: half a unit of the result (2^-8 of it at most for bf16, 2^-11 for f16), and 2^-14 of the terms (1 + lambda) |v| for what
is held in 32 bits (scores do not matter here; products, sums, reciprocals and the norm do). With lambda 0.9 a divisor
of unrounded probabilities is off by up to 2^-8 (1 + lambda) |v| in bf16, over ten times that tolerance. A large eps keeps the
norm from dividing a common factor out.
"""
import pytest
import torch

import tsn
from test_gpu_diff_attn import DT, make
from test_gpu_diff_attn import dev  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("typ", ["f16", "bf16"])
@pytest.mark.parametrize("d", [32, 64])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("Sq,Sk", [(1, 60), (4, 700), (2, 20000), (130, 130), (100, 500), (64, 6000)])
def test_values_that_are_alike(dev, Sq, Sk, causal, d, typ):  # noqa: F811
    q, k, v, _, w = make(3 * Sq + Sk, typ, d, 2, Sq, Sk, 4, 2, gain=2.5)   # few keys carry a row, found one after another
    v[:] = v[:, :1]
    zero = [torch.zeros(d, device="cuda")] * 4
    lam, eps = 0.9, 1e4
    op = tsn.DiffAttention(dev, d, *zero, lambda_init=lam, norm_weight=w, eps=eps)
    out = torch.full_like(q, float("nan"))
    op(q, k, v, out, causal=causal)
    dev.commit()
    x = v[:, :1].double().repeat_interleave(2, 2)                     # [B, 1, H, 2 d]
    o = (1 - lam) * x
    g = (1 - lam) * w.double() / (o.square().mean(-1, keepdim=True) + eps).sqrt()
    tol = (o * g).abs() * {"bf16": 2.0 ** -8, "f16": 2.0 ** -11}[typ] + (1 + lam) * x.abs() * g.abs() * 2.0 ** -14
    tol = tol + (2.0 ** -25 if typ == "f16" else 0.0)
    err = (out.double() - o * g).abs()
    assert out.dtype is DT[typ] and bool((err <= tol).all()), float((err / tol).max())
