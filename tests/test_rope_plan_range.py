"""The rotary plan refuses turns per position that are no finite number (a small theta or a large scale overflows), which have no
fraction to hold. Host only."""
import ctypes as C

import pytest

import tsn


def plan(pairs, theta, scale):
    n, p = len(pairs), tsn.RopePlan()
    tsn.check(tsn.lib().tsn_rope_plan(64, n, (C.c_uint32 * n)(*pairs), (C.c_double * n)(*theta), (C.c_double * n)(*scale), 0, C.byref(p)))
    return p


@pytest.mark.parametrize("theta,scale", [(1e-300, 1e300), (1e-300, -1e25), (5e-324, 1.0)])
def test_turns_that_overflow(theta, scale):
    with pytest.raises(tsn.TsnError) as e:
        plan((8, 24), (1e4, theta), (1.0, scale))
    assert e.value.code == 1 and "tsn_rope_plan" in str(e.value)


@pytest.mark.parametrize("theta,scale", [(1e-300, 1.0), (1e300, 1e300), (1e4, 0.0)])
def test_turns_that_are_finite(theta, scale):
    assert plan((8, 24), (1e4, theta), (1.0, scale)).P == 32
