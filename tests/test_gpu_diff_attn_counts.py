"""Differential attention: counts whose product passes 32 bits are refused by name, before any launch. The operands' addresses
are of a small buffer that is never reached."""
import pytest
import torch

import tsn

pytestmark = pytest.mark.gpu


# groups of rows x sequences x kv heads: 2^32 twice, which 32 bits would hold as 0, then numbers on either side
@pytest.mark.parametrize("B,H,Sq", [(32768, 32768, 25), (32768, 32768, 512), (65535, 65535, 9), (65535, 65535, 1)])
def test_products_past_32_bits(B, H, Sq):
    dev = tsn.Device(0, stream=torch.cuda.current_stream().cuda_stream)
    small = torch.zeros(1024, dtype=torch.float16, device="cuda")
    lam = torch.zeros(64, device="cuda")
    heads = tsn.Heads(p=small.data_ptr(), sb=128 * H, ss=128, sh=128)
    p = lam.data_ptr()
    a = tsn.DiffAttnArgs(B=B, Sq=Sq, Sk=16, H=H, Hk=H, d=64, type=1, lambda_init=0.4, eps=1e-5, q=heads, k=heads, v=heads, out=heads,
                         lq1=p, lk1=p, lq2=p, lk2=p)
    assert tsn.lib().tsn_diff_attn(dev.h, a) == 1
    assert b"too many query rows" in tsn.lib().tsn_last_error()
    dev.commit()
    dev.close()
