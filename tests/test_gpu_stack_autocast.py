"""PoMStack.train_forward under autocast to bfloat16: float32 tokens pass the residual path unrounded, in both directions."""
import pytest
import torch

from oracle import pom_oracle as O
from tests.helpers import BF16_TOL
from tests.test_gpu_stack_train import make, reference, rel

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kw", [dict(norm=True, bias=True), dict(norm=True, activation="silu"), dict()])
def test_tokens_pass_blocks_that_add_nothing(kw):
    stack, _ = make(64, 2, torch.float32, **kw)
    with torch.no_grad():
        for m in [*stack.ffn_out, *(m.ag_proj for m in stack.mixers)]:
            for p in m.parameters():
                p.zero_()
    x, gy = torch.randn(2, 96, 64, device="cuda").requires_grad_(True), torch.randn(2, 96, 64, device="cuda")
    with torch.autocast("cuda", torch.bfloat16):
        y = stack.train_forward(x, "causal")
    assert y.dtype == torch.float32 and torch.equal(y, x)
    dx, = torch.autograd.grad(y, x, gy)
    assert dx.dtype == torch.float32 and torch.equal(dx, gy)


def test_small_branches_beside_large_tokens():
    """Tokens near 1000, whose bf16 steps are 4 to 8 wide, and branches of size 1: the branches keep the accuracy that the
    products have, because nothing rounds the sum (2^-24 of 1000 is 6e-5)."""
    stack, params = make(64, 2, torch.float32, norm=True, bias=True)
    x = torch.randn(2, 96, 64) * 3 + 1000
    want = reference({k: v.double() for k, v in params.items()}, stack, x.double(), "causal") - x.double()
    with torch.autocast("cuda", torch.bfloat16), torch.no_grad():
        y = stack.train_forward(x.cuda(), "causal")
    assert y.dtype == torch.float32
    assert rel(y.double() - x.cuda().double(), want) <= 3 * BF16_TOL


def test_other_types_as_they_were():
    stack, _ = make(64, 2, torch.float32, norm=True, bias=True)
    x = O.bf16_round(torch.randn(2, 96, 64)).cuda()
    with torch.no_grad():
        assert stack.train_forward(x, "causal").dtype == torch.float32
        with torch.autocast("cuda", torch.bfloat16):
            assert stack.train_forward(x.bfloat16(), "causal").dtype == torch.bfloat16
