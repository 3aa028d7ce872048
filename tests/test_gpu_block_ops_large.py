"""Layer norm, linear and several-axis rotary operators on tensors of more than 2^31 elements: offsets in 64 bits, seen at the
last rows, in both directions."""
import pytest
import torch

from pom_b200.operators import apply_rope_axes, layer_norm, linear, precompute_freqs_axes
from tests.test_gpu_block_ops import BF, E, act_reference, norm_reference, rand, rope_reference, within

pytestmark = pytest.mark.gpu

TAIL = 70


@pytest.fixture(autouse=True)
def room():
    free, _ = torch.cuda.mem_get_info()
    if free < 60 << 30:
        pytest.skip("needs 60 GB of device memory")
    yield
    torch.cuda.empty_cache()


def large(rows, width, seed):
    return torch.empty(rows, width, device="cuda", dtype=BF).normal_(generator=torch.Generator(device="cuda").manual_seed(seed))


def test_layer_norm():
    M, D = 1_864_200, 1152
    assert M * D > 2 ** 31
    x, w, b, dy = large(M, D, 1).requires_grad_(True), rand(D, dtype=BF, seed=2, shift=1.0), rand(D, dtype=BF, seed=3), large(M, D, 4)
    y = layer_norm(x, w, b)
    dx, = torch.autograd.grad(y, x, dy)
    want, slack = norm_reference(x[-TAIL:], w, b, 1e-5, dy[-TAIL:])
    within(y[-TAIL:], want[0], slack[0], "y")
    within(dx[-TAIL:], want[1], slack[1], "dx")


def test_linear():
    M, K, N = 466_100, 64, 4608
    assert M * N > 2 ** 31
    x, w, b, r = large(M, K, 1).requires_grad_(True), rand(N, K, dtype=BF, seed=2, scale=K ** -0.5), rand(N, dtype=BF, seed=3), large(M, N, 4)
    y = linear(x, w, b, activation="silu", residual=r)
    dy = large(M, N, 5)
    dx, = torch.autograd.grad(y, x, dy)
    xd, wd, g = x[-TAIL:].detach().double(), w.double(), dy[-TAIL:].double()
    z = xd @ wd.t() + b.double()
    ze = 2 * (K + 8) * E * (xd.abs() @ wd.abs().t() + b.double().abs())
    a, s = act_reference(z, "silu")
    want = a + r[-TAIL:].double()
    within(y[-TAIL:], want, 1.13 * ze + 16 * E * (z.abs() + 1) + E * (a.abs() + want.abs()), "y")
    h = 2.0 ** -8
    se = 0.8 * (ze + h * z.abs()) + 16 * E * (z.abs() + 1)
    dz = g * s
    stored = g.abs() * se + h * dz.abs()
    within(dx[-TAIL:], dz @ wd, stored @ wd.abs() + 2 * (N + 8) * E * (dz.abs() @ wd.abs()), "dx")


def test_linear_weight_of_few_rows():
    M, K, N = 3, 4096, 524_400
    assert N * K > 2 ** 31
    x, w = rand(M, K, dtype=BF, seed=1), large(N, K, 2)
    y = linear(x, w)
    xd, wd = x.double(), w[-TAIL:].double()
    want = xd @ wd.t()
    within(y[:, -TAIL:], want, 2 * (K + 8) * E * (xd.abs() @ wd.abs().t()) + E * want.abs(), "y")


@pytest.mark.parametrize("heads", [0, 16])
def test_rope_axes(heads):
    N, D = (932_100, 2304) if not heads else (1_864_200, 72)
    x = large(N, D * max(1, heads), 1).view(1, N, *((heads,) if heads else ()), D).requires_grad_(True)
    assert x.numel() > 2 ** 31
    pairs = (384, 384, 384) if not heads else (8, 12, 16)
    tables = [(c, s) for c, s in precompute_freqs_axes(pairs, (100, 100, 200), device="cuda")]
    i = torch.arange(N, device="cuda")
    pos = torch.stack([i // 20000 % 100, i // 200 % 100, i % 200], -1)
    y = apply_rope_axes(x, pos, tables)
    dx, = torch.autograd.grad(y, x, x.detach())
    tail = x[:, -TAIL:].detach()
    within(y[:, -TAIL:].detach(), *rope_reference(tail, pos[-TAIL:], tables, False), "y")
    within(dx[:, -TAIL:], *rope_reference(tail, pos[-TAIL:], tables, True), "dx")
