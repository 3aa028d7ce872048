"""Few-row products of the linear operator: every number of rows, widths that fill a block's columns and that do not, with and
without bias and residual.  What is absent (a bias, a residual, rows and columns of a tile) is never read."""
import pytest
import torch

from pom_b200.operators import linear
from tests.test_gpu_block_ops import BF, E, F32, act_reference, rand, within

pytestmark = pytest.mark.gpu


def check(x, w, b, r, act):
    with torch.no_grad():
        y = linear(x, w, b, activation=act, residual=r)
    xd, wd = x.double(), w.double()
    z, ze = xd @ wd.t(), xd.abs() @ wd.abs().t()
    if b is not None:
        z, ze = z + b.double(), ze + b.double().abs()
    ze = 2 * (x.shape[1] + 8) * E * ze
    want = act_reference(z, act)[0]
    slack = 1.13 * ze + (0 if act is None else 16 * E * (z.abs() + 1)) + E * want.abs()
    if r is not None:
        want = want + r.double()
    within(y, want, slack + E * want.abs(), f"{tuple(x.shape)} -> {w.shape[0]}, bias {b is not None}, residual {r is not None}")


@pytest.mark.parametrize("N", [8, 13, 200, 2360, 2368, 2369, 2376, 4056, 4064])
@pytest.mark.parametrize("K", [8, 136, 1016, 2048])
def test_bf16(K, N):
    w, b = rand(N, K, dtype=BF, seed=1, scale=K ** -0.5), rand(N, seed=2)
    for M in (20, *range(1, 34)):
        x, r = rand(M, K, dtype=BF, seed=3 + M), rand(M, N, dtype=BF, seed=4)
        for bias in (None, b if M % 2 else b.to(BF)):
            for res in (None, r):
                check(x, w, bias, res, ("relu", None, "gelu", "silu")[M % 4])


@pytest.mark.parametrize("N", [1, 7, 8, 300, 2049])
@pytest.mark.parametrize("K", [4, 132, 1016])
def test_float32(K, N):
    w, b = rand(N, K, seed=1, scale=K ** -0.5), rand(N, seed=2)
    for M in range(1, 18):
        x, r = rand(M, K, seed=3 + M), rand(M, N, seed=4)
        for bias in (None, b):
            for res in (None, r):
                check(x, w, bias, res, ("relu", None, "gelu", "silu")[M % 4])


def test_operands_at_the_end_of_their_memory():
    """x, weight, bias and residual end with the memory that the allocator has for them: nothing behind them is read."""
    torch.cuda.empty_cache()
    for M, K, N, dtype in ((20, 1016, 4056, BF), (3, 1016, 4056, BF), (20, 136, 200, BF), (5, 132, 300, F32), (11, 1016, 2049, F32)):
        item = 2 if dtype == BF else 4

        def at_end(*shape):  # 32 MB are a piece of memory of their own
            n = torch.Size(shape).numel()
            whole = torch.empty((32 << 20) // item, device="cuda", dtype=dtype)
            t = whole[whole.numel() - (n + 7) // 8 * 8:][:n].view(shape)
            return t.copy_(rand(*shape, dtype=dtype, seed=n))

        x, w, b, r = at_end(M, K), at_end(N, K), at_end(N), at_end(M, N)
        for bias in (None, b):
            for res in (None, r):
                check(x, w, bias, res, "relu")
