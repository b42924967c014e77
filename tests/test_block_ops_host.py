"""The transformer-block operators' host side, without a GPU: struct layouts of the binding, the rotary plan's
fractions, and refusals that come before any device work."""
import ctypes as C
import math
import os
import subprocess
from fractions import Fraction

import pytest

import tsn

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
STRUCTS = {"tsn_rows": tsn.Rows, "tsn_heads": tsn.Heads, "tsn_block_norm_args": tsn.BlockNormArgs,
           "tsn_rope_plan_t": tsn.RopePlan, "tsn_rope_args": tsn.RopeArgs, "tsn_diff_attn_args": tsn.DiffAttnArgs}


def test_binding_has_the_headers_layouts(tmp_path):
    lines = []
    for name, cls in STRUCTS.items():
        lines.append(f'printf("{name} %zu", sizeof({name}));')
        lines += [f'printf(" %zu", offsetof({name}, {f[0]}));' for f in cls._fields_]
        lines.append('printf("\\n");')
    src = tmp_path / "layout.c"
    src.write_text('#include <stdio.h>\n#include "tsn.h"\nint main(void) {\n' + "\n".join(lines) + "\nreturn 0;\n}\n")
    exe = str(tmp_path / "layout")
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", exe], check=True)
    for line in subprocess.run([exe], check=True, capture_output=True, text=True).stdout.splitlines():
        name, *numbers = line.split()
        cls = STRUCTS[name]
        assert [int(n) for n in numbers] == [C.sizeof(cls)] + [getattr(cls, f[0]).offset for f in cls._fields_], name


def plan(D, pairs, theta, scale, layout=0):
    n = len(pairs)
    p = tsn.RopePlan()
    tsn.check(tsn.lib().tsn_rope_plan(D, n, (C.c_uint32 * n)(*pairs), (C.c_double * n)(*theta), (C.c_double * n)(*scale),
                                      layout, C.byref(p)))
    return p


@pytest.mark.parametrize("D,pairs,theta,scale", [(64, (8, 12, 12), (1e4,) * 3, (1.0,) * 3), (256, (128,), (5e5,), (1.0,)),
                                                 (64, (8, 8, 8, 8), (100.0, 1e4, 1e6, 2.0), (0.25, -1.0, 40.0, 1e-3)),
                                                 (6, (0, 3), (1e4, 1e4), (1.0, 0.0))])
def test_plan_holds_each_pairs_turns(D, pairs, theta, scale):
    p = plan(D, pairs, theta, scale)
    assert (p.D, p.axes, p.P) == (D, len(pairs), sum(pairs))
    j = 0
    for a, n in enumerate(pairs):
        for i in range(n):
            turns = scale[a] * theta[a] ** (-i / n) / (2 * math.pi)
            held = Fraction(p.turn[j], 2 ** 64)
            # the double behind it has 53 bits; a turn more or less is the same angle
            off = abs(held - Fraction(turns) % 1)
            assert min(off, 1 - off) <= Fraction(abs(turns)) / 2 ** 50 + Fraction(1, 2 ** 53)
            assert p.axis[j] == a
            j += 1


def test_plan_refusals():
    for D, pairs, theta, scale in ((63, (8,), (1e4,), (1.0,)), (0, (0,), (1e4,), (1.0,)), (64, (33,), (1e4,), (1.0,)),
                                   (64, (2 ** 32 - 1, 2), (1e4,) * 2, (1.0,) * 2), (64, (8,), (-1.0,), (1.0,)),
                                   (64, (8,), (1e4,), (math.nan,)), (64, (1,) * 5, (1e4,) * 5, (1.0,) * 5)):
        with pytest.raises(tsn.TsnError) as e:
            plan(D, pairs, theta, scale)
        assert e.value.code == 1
    with pytest.raises(tsn.TsnError):
        plan(64, (8,), (1e4,), (1.0,), layout=2)
    assert tsn.lib().tsn_rope_plan(64, 1, None, None, None, 0, None) == 1


def test_null_handles():
    L = tsn.lib()
    assert L.tsn_block_norm(None, tsn.BlockNormArgs()) == 1
    assert L.tsn_rope_axes(None, tsn.RopePlan(), tsn.RopeArgs()) == 1
    assert L.tsn_diff_attn(None, tsn.DiffAttnArgs()) == 1


def test_binding_without_torch():
    """The rest of the binding does not import torch."""
    code = "import sys; sys.path.insert(0, %r); import tsn; tsn.lib(); assert 'torch' not in sys.modules" % os.path.join(
        ROOT, "thinksound-native_b200")
    subprocess.run(["python3", "-c", code], check=True)


def test_tensors_of_another_gpu_are_refused():
    """An operator's tensors lie on its handle's GPU: not on another one, not in host memory."""
    from tsn import block_ops

    class Dev:
        ordinal = 1

    class On:
        def __init__(self, gpu):
            self.gpu = gpu

        def get_device(self):
            return self.gpu

    block_ops._here(Dev, ("x", On(1)), ("y", None))
    for gpu in (0, 2, -1):
        with pytest.raises(ValueError, match="y must be a CUDA tensor on GPU 1"):
            block_ops._here(Dev, ("x", On(1)), ("y", On(gpu)))
