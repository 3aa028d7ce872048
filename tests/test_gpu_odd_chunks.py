"""Widths whose tiles hold an odd number of 32-column chunks, over so many tokens that every block walks several tiles: the two
staging blocks of a warp's stores alternate anew in every tile, so a tile begins on the block that the one before ended on."""
import pytest
import torch

from oracle import pom_oracle as O
from pom_b200 import PoM, PoMRoPE
from tests.helpers import BF16_TOL, assert_close, assert_status_clean

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dim", [80, 176])  # 160 and 352 projected channels: 5 and 11 chunks
@pytest.mark.parametrize("cls, kw", [(PoM, {}), (PoMRoPE, dict(max_seq_len=32768))])
def test_many_tiles_of_odd_width(cls, kw, dim):
    torch.manual_seed(7)
    mod = cls(dim, 2, 2, **kw)
    with torch.no_grad():
        mod.po_coeff.copy_(torch.randn_like(mod.po_coeff) * 0.3)
        for p in mod.parameters():
            p.copy_(O.bf16_round(p))
    x = O.bf16_round(torch.randn(2, 32768, dim)).cuda()
    mod = mod.cuda()
    with torch.no_grad():
        want = mod(x)  # float32
    for p in mod.parameters():
        p.data = p.data.bfloat16()
    xb = x.bfloat16().requires_grad_(True)
    gy = O.bf16_round(torch.randn(2, 32768, dim)).cuda().bfloat16()
    with torch.no_grad():
        infer = mod(xb)
    assert_close(infer, want, BF16_TOL, "y without a gradient")
    first = None
    for _ in range(3):
        y = mod(xb)
        dx, = torch.autograd.grad(y, xb, gy)
        assert_close(y.detach(), want, BF16_TOL, "y")
        first = (y, dx) if first is None else first
        assert_close(dx, first[1], BF16_TOL, "dx again")
    assert_status_clean()
