"""Activations of the linear operator and their slopes far from 0: through an identity weight, where the products add nothing,
so that every value is the activation's own."""
import math

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


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("rows", [24, 600])
def test_gelu_keeps_its_digits_in_the_tail(rows, dtype):
    """Relative to the value, not to 1.  z Phi(z) and Phi(z) + z phi(z), with two kinds of error: the stored value is rounded
    (half a step: 2^-8 or 2^-24 of it), and the terms are formed with a relative error of at most 2^-15 in bf16 (the
    coefficients 2^-18; exp(-z^2 / 2): three roundings of z^2 / 2 <= 83, 83 * 3 * 2^-24 = 2^-16; some 2^-22 beside them) and of
    (1.5 z^2 + 16) 2^-24 in float32 (the same three roundings, and four times four units of erfc, exp and the products)."""
    h = 2.0 ** -8 if dtype == BF else 2.0 ** -24
    z = torch.cat([torch.linspace(-12.9, -0.01, 480), torch.linspace(0.01, 12.9, 120)]).cuda().to(dtype)
    got = [through(part, "gelu") for part in z.split(rows)]
    y, slope = (torch.cat([g[i] for g in got]).double() for i in (0, 1))
    z = z.double()
    phi = 0.5 * torch.special.erfc(-z / math.sqrt(2))
    pdf = z.abs() * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    formed = 2.0 ** -15 if dtype == BF else (1.5 * z * z + 16) * 2.0 ** -24
    want, want_slope = z * phi, phi + z.sign() * pdf
    for name, a, b, size in (("y", y, want, want.abs()), ("slope", slope, want_slope, phi + pdf)):
        off = (a - b).abs() - (h * b.abs() + formed * size)
        i = int(off.argmax())
        assert off[i] <= 0, (name, z[i].item(), a[i].item(), b[i].item())
