"""A plan that tsn_rope_plan did not make is refused before anything is read past it: no count of pairs wraps around the check."""
import ctypes as C

import pytest
import torch

import tsn

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("change", [dict(P=2 ** 31), dict(P=2 ** 31 + 5), dict(P=33), dict(P=2 ** 32 - 1), dict(D=0), dict(D=63), dict(D=258),
                                    dict(axes=0), dict(axes=5)])
def test_plans_that_are_none(change):
    dev = tsn.Device(0, stream=torch.cuda.current_stream().cuda_stream)
    plan = tsn.RopePlan()
    tsn.check(tsn.lib().tsn_rope_plan(64, 1, (C.c_uint32 * 1)(32), (C.c_double * 1)(1e4), (C.c_double * 1)(1.0), 0, C.byref(plan)))
    x, pos = torch.zeros(1, 1, 1, 256, device="cuda"), torch.zeros(1, 1, dtype=torch.int32, device="cuda")
    heads = tsn.Heads(p=x.data_ptr(), sb=256, ss=256, sh=256)
    a = tsn.RopeArgs(B=1, S=1, Hq=1, type=0, eps=1e-6, q=heads, q_out=heads, pos=pos.data_ptr(), pos_ss=1)
    assert tsn.lib().tsn_rope_axes(dev.h, plan, a) == 0
    for name, value in change.items():
        setattr(plan, name, value)
    assert tsn.lib().tsn_rope_axes(dev.h, plan, a) == 1
    assert b"not a plan" in tsn.lib().tsn_last_error()
    dev.commit()
    dev.close()
