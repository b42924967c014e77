"""Block norm of rows that start at pairs of elements but not at 16 bytes: an even C, or a pitch or start that is."""
import pytest
import torch

from test_gpu_block_norm import DT, check_case, dev, make  # noqa: F401

pytestmark = pytest.mark.gpu
TYPES = [("f32", "f32"), ("f16", "f16"), ("bf16", "bf16"), ("f16", "f32"), ("bf16", "f32")]


@pytest.mark.parametrize("typ,xtyp", TYPES)
@pytest.mark.parametrize("C", [2, 6, 62, 66, 130, 1022, 1462, 2050, 4098, 8190, 8194, 16382])
def test_even_lengths(dev, typ, xtyp, C):  # noqa: F811
    x, y, gate, shift, scale, w, r = make(C, 3, 5, C, typ, xtyp)
    check_case(dev, x, y, gate, shift, scale, w, typ, xtyp, "rms", "layer", residual_scale=r)
    check_case(dev, x, None, None, shift, scale, w, typ if xtyp == typ else xtyp, xtyp, "none", "rms") if typ == xtyp else None


@pytest.mark.parametrize("typ,xtyp", TYPES)
@pytest.mark.parametrize("rows", [1, 149, 3000])
def test_rows(dev, typ, xtyp, rows):  # noqa: F811
    x, y, gate, shift, scale, w, r = make(rows, 2, rows, 462, typ, xtyp, gate="token", mod="token")
    check_case(dev, x, y, gate, shift, scale, w, typ, xtyp, "layer", "rms", residual_scale=0.5, gate_tanh=typ != "bf16")


@pytest.mark.parametrize("typ", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("pad,skip", [(2, 0), (0, 2), (6, 4), (1, 0), (0, 1)])
def test_pitch_and_start(dev, typ, pad, skip):  # noqa: F811
    """C itself is a multiple of 16 bytes; the rows' distance or first element is not (odd ones take the elements' path)."""
    C = 1024
    x, y, gate, shift, scale, w, r = make(pad * 8 + skip, 2, 9, C, typ, typ)
    base = torch.full((2, 9, C + pad + skip), float("nan"), dtype=DT[typ], device="cuda")
    base[..., skip:skip + C] = x
    check_case(dev, base[..., skip:skip + C], y, gate, shift, scale, w, typ, typ, "rms", "layer")
