"""Layer norm and linear with every combination of absent operands, at sizes where blocks walk several rows or tiles and leave parts
of them out."""
import pytest
import torch

from tests.test_gpu_block_ops import BF, F32, linear_check, linear_inputs, norm_check, rand

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("D", [96, 161, 1152, 1288, 2049, 4104])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_layer_norm(D, dtype):
    for M in (1, 13, 8_000_000 // D):  # the last: more rows than a block's share
        x, dy = rand(M, D, dtype=dtype, seed=1, shift=0.3), rand(M, D, dtype=dtype, seed=2)
        for w, b in ((None, None), (rand(D, dtype=dtype, seed=3, shift=1.0), None), (rand(D, seed=3, shift=1.0), rand(D, seed=4))):
            norm_check(x, w, b, dy, label=f"{M} ")


@pytest.mark.parametrize("M, K, N", [(34, 1016, 4056), (65, 3080, 1096), (385, 136, 520), (1000, 2056, 264), (3000, 264, 1160)])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_linear(M, K, N, dtype):
    x, w, b, r, dy = linear_inputs(M, K, N, dtype, seed=7)
    for act in (None, "relu", "gelu"):
        for bias in (None, b, b.float()):
            for res in (None, r):
                linear_check(x, w, bias, res, act, dy, label=f"{act}, bias {bias is not None}, residual {res is not None}: ")
