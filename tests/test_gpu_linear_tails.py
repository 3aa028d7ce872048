"""Activations of the linear operator and their slopes far from 0: through an identity weight, where the products add nothing,
so that every value is the activation's own."""
import pytest
import torch

from pom_b200.operators import linear

pytestmark = pytest.mark.gpu

BF, F32 = torch.bfloat16, torch.float32
ACTS = ["gelu", "gelu_tanh", "silu", "relu"]


def through(z, act, width=8):
    """act(z) and its slope for a vector z: z is the first column of the tokens, the weight an identity."""
    x = torch.zeros(len(z), width, device="cuda", dtype=z.dtype)
    x[:, 0] = z
    x.requires_grad_(True)
    y = linear(x, torch.eye(width, device="cuda", dtype=z.dtype), activation=act)
    g = torch.zeros_like(y)
    g[:, 0] = 1
    dx, = torch.autograd.grad(y, x, g)
    return y.detach()[:, 0], dx[:, 0], dx[:, 1:]


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("dtype, width", [(BF, 8), (F32, 8), (F32, 7)])
@pytest.mark.parametrize("rows", [12, 120])
def test_slopes_of_values_up_to_the_largest(rows, dtype, width, act):
    """Every finite value beyond 1e4 has the slope 1 or 0 exactly: nothing overflows into 0 * infinity."""
    z = torch.tensor([s * m for m in (1e4, 3e9, 2e13, 1e19, 1e25, 3e38) for s in (1.0, -1.0)], device="cuda").to(dtype)
    z = z.repeat(rows // 12)
    y, slope, others = through(z, act, width)
    assert torch.equal(slope, (z > 0).to(dtype))
    assert torch.equal(y, torch.where(z > 0, z, torch.zeros_like(z)))
    assert not others.any()  # the columns beside it stay free of NaN
