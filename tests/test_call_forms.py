"""The form of a call's tensors (tsn_form_take through tsn.block_ops): what has the form of the call before skips the
checks, anything else goes through them, and the addresses are those of the call's own tensors. Host only."""
import ctypes as C
import os
import subprocess

import pytest
import torch

import tsn
from tsn import block_ops

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
NAMES = ("x", "y", "gate", "shift", "scale", "x_out", "h")


class Host:
    """A handle whose tensors lie in host memory."""
    ordinal = -1
    h = C.c_void_p(0)


@pytest.fixture
def norm():
    """A norm whose launches are counted checks: call(**tensors) returns whether the call was checked."""
    op = block_ops.BlockNorm(Host, 16, "rms", "rms")
    checked, check = [], op._check
    op._check = lambda *t: (checked.append(1), check(*t))
    op._call = lambda dev, args: 0

    def call(**tensors):
        checked.clear()
        op(**tensors)
        for name, view in zip(NAMES, op._views):
            t = tensors.get(name)
            assert (view.p or 0) == (0 if t is None else t.data_ptr()), name
        return bool(checked)

    call.op = op
    return call


def test_layouts(tmp_path):
    structs = {"tsn_form": tsn.Form, "tsn_form_tensor": tsn.FormTensor}
    lines = []
    for name, cls in structs.items():
        lines.append(f'printf("{name} %zu", sizeof({name}));')
        lines += [f'printf(" %zu", offsetof({name}, {f[0]}));' for f in cls._fields_]
        lines.append('printf("\\n");')
    src = tmp_path / "layout.c"
    src.write_text('#include <stddef.h>\n#include <stdio.h>\n#include "tsn.h"\nint main(void) {\n' + "\n".join(lines)
                   + "\nreturn 0;\n}\n")
    exe = str(tmp_path / "layout")
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", exe], check=True)
    for line in subprocess.run([exe], check=True, capture_output=True, text=True).stdout.splitlines():
        name, *numbers = line.split()
        cls = structs[name]
        assert [int(n) for n in numbers] == [C.sizeof(cls)] + [getattr(cls, f[0]).offset for f in cls._fields_], name


def test_same_form_is_checked_once(norm):
    assert block_ops._VIEW
    base = torch.zeros(4, 6, 32)
    x, y, gate = base[:, :3, :16], base[:, 3:, 16:], torch.zeros(1, 1, 16)
    assert norm(x=x, y=y, gate=gate, x_out=x)
    assert not norm(x=x, y=y, gate=gate, x_out=x)
    other = torch.zeros(4, 6, 32)
    assert not norm(x=other[:, 3:, :16], y=other[:, :3, :16], gate=gate.clone(), x_out=other[:, 3:, 16:])


def other_forms():
    base = torch.zeros(4, 3, 16)
    yield "shape", base[:2]
    yield "tokens", base[:, :2]
    yield "strides", torch.zeros(4, 6, 16)[:, ::2]
    yield "batch stride", torch.zeros(8, 3, 16)[::2]
    yield "type", base.half()
    yield "parameter", torch.nn.Parameter(base.clone(), requires_grad=False)


@pytest.mark.parametrize("name,t", list(other_forms()), ids=[n for n, _ in other_forms()])
def test_another_form_is_checked(norm, name, t):
    x = torch.zeros(4, 3, 16)
    assert norm(x=x, x_out=x) and not norm(x=x, x_out=x)
    assert norm(x=t, x_out=torch.empty_like(t)) or name == "parameter"
    assert norm(x=x, x_out=x) or name == "parameter"
    assert not norm(x=x, x_out=x)


def test_absent_and_present(norm):
    x = torch.zeros(2, 3, 16)
    for tensors in (dict(x=x, x_out=x), dict(x=x, y=x, x_out=x), dict(x=x, h=x), dict(x=x, y=x, h=x, shift=x)):
        assert norm(**tensors) and not norm(**tensors)


def test_no_tensors_bytes(norm):
    empty = torch.zeros(0, 3, 16)
    assert norm(x=empty, x_out=empty) and not norm(x=empty, x_out=empty)


def test_gradients_and_offsets(norm):
    x = torch.zeros(2, 3, 16)
    assert norm(x=x, x_out=x)
    assert not norm(x=x.clone().requires_grad_(), x_out=x)
    assert not norm(x=torch.zeros(101)[5:].as_strided((2, 3, 16), (48, 16, 1)), x_out=x)


@pytest.mark.parametrize("bad", [torch.eye(16).to_sparse(), "x", 3, torch.zeros(3, 16), torch.zeros(2, 2, 2, 2, 16),
                                 torch.empty(2, 3, 16, device="meta")], ids=["sparse", "text", "number", "2d", "5d", "meta"])
def test_what_is_no_tensor_of_a_call_is_refused(norm, bad):
    x = torch.zeros(2, 3, 16)
    assert norm(x=x, x_out=x)
    with pytest.raises((ValueError, TypeError, AttributeError)):
        norm.op(bad, x_out=x)
    assert norm(x=x, x_out=x)   # a refused call leaves no form behind
    with pytest.raises((ValueError, TypeError, AttributeError)):
        norm.op(x, x_out=bad)
    assert norm(x=x, x_out=x)


def test_every_operator_sets_its_addresses():
    lam = torch.zeros(32)
    op = block_ops.DiffAttention(Host, 32, lam, lam, lam, lam, 0.2)
    op._call = lambda dev, args: 0
    rope = block_ops.RopeAxes(Host, 64, (8, 8))
    rope._call = lambda dev, plan, args: 0
    for _ in range(2):
        for _ in range(2):
            q, k, v, out = (torch.zeros(2, 5, 4, 64, dtype=torch.float16) for _ in range(4))
            n, mask = torch.zeros(2, dtype=torch.int32), torch.zeros(2, 5, dtype=torch.bool)
            op(q, k, v, out, key_len=n, key_mask=mask)
            a = op._a
            assert [a.q.p, a.k.p, a.v.p, a.out.p, a.key_len, a.key_mask] == [t.data_ptr() for t in (q, k, v, out, n, mask)]
            pos = torch.zeros(5, 2, dtype=torch.int32)
            rope(q, k, pos)
            r = rope._a
            assert [r.q.p, r.k.p, r.q_out.p, r.k_out.p, r.pos] == [t.data_ptr() for t in (q, k, q, k, pos)]
        op(q, k, v, out)
        assert op._a.key_len is None and op._a.key_mask is None
        rope(q, None, pos, q_out=out)
        assert [r.q.p, r.k.p, r.q_out.p, r.k_out.p] == [q.data_ptr(), None, out.data_ptr(), None]
