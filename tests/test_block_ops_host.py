"""Layer norm, linear and several-axis rotary operators: what needs no GPU — refusals, the argument structs, the tables."""
import ctypes
import os
import subprocess
import tempfile

import pytest
import torch

from pom_b200 import _abi, ops
from pom_b200.operators import apply_rope_axes, layer_norm, linear, precompute_freqs_axes
from pom_b200.pom_rope import precompute_freqs_2d

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def t(*shape, dtype=torch.float32):
    return torch.zeros(*shape, dtype=dtype)


def test_struct_sizes_match_the_c_compiler():
    structs = {"pom_layer_norm_args": _abi.LayerNormArgs, "pom_linear_args": _abi.LinearArgs,
               "pom_rope_axes_args": _abi.RopeAxesArgs}
    src = '#include <stdio.h>\n#include "pom_b200.h"\nint main(void){' + "".join(
        f'printf("{n} %zu\\n", sizeof({n}));' for n in structs) + "return 0;}\n"
    with tempfile.TemporaryDirectory() as d:
        c, exe = os.path.join(d, "s.c"), os.path.join(d, "s")
        with open(c, "w") as f:
            f.write(src)
        subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), c, "-o", exe], check=True)
        out = subprocess.run([exe], check=True, capture_output=True, text=True).stdout
    for line in out.strip().splitlines():
        name, size = line.split()
        assert ctypes.sizeof(structs[name]) == int(size), name


@pytest.mark.parametrize("call, error", [
    (lambda: layer_norm(t(4, 8, dtype=torch.float16)), TypeError),
    (lambda: layer_norm([1.0]), TypeError),
    (lambda: layer_norm(t(4, 0)), ValueError),
    (lambda: layer_norm(torch.tensor(1.0)), ValueError),
    (lambda: layer_norm(t(4, 8), t(7)), ValueError),
    (lambda: layer_norm(t(4, 8), t(1, 8)), ValueError),
    (lambda: layer_norm(t(4, 8), t(8), t(9)), ValueError),
    (lambda: layer_norm(t(4, 8), None, t(8)), ValueError),
    (lambda: layer_norm(t(4, 8), t(8, dtype=torch.int64)), TypeError),
    (lambda: layer_norm(t(4, 8), t(8)), RuntimeError),  # not on a GPU
    (lambda: linear(t(4, 8), t(3, 7)), ValueError),
    (lambda: linear(t(4, 8), t(8)), ValueError),
    (lambda: linear(t(4, 0), t(3, 0)), ValueError),
    (lambda: linear(t(4, 8), t(3, 8), t(4)), ValueError),
    (lambda: linear(t(4, 8), t(3, 8), t(3, 1)), ValueError),
    (lambda: linear(t(4, 8), t(3, 8), activation="tanh"), ValueError),
    (lambda: linear(t(4, 8), t(3, 8), residual=t(3)), ValueError),
    (lambda: linear(t(4, 8), t(3, 8), residual=t(1, 3)), ValueError),
    (lambda: linear(t(4, 8), t(3, 8, dtype=torch.bfloat16)), TypeError),
    (lambda: linear(t(4, 8), t(3, 8), residual=t(4, 3, dtype=torch.bfloat16)), TypeError),
    (lambda: linear(t(4, 8, dtype=torch.float64), t(3, 8)), TypeError),
    (lambda: linear(t(4, 8), t(3, 8)), RuntimeError),
    (lambda: apply_rope_axes(t(4, 8), t(4, 1, dtype=torch.int64), [(t(9, 2), t(9, 2))]), ValueError),
    (lambda: apply_rope_axes(t(1, 4, 8), t(4, 0, dtype=torch.int64), []), ValueError),
    (lambda: apply_rope_axes(t(1, 4, 80), t(4, 5, dtype=torch.int64), [(t(9, 2), t(9, 2))] * 5), ValueError),
    (lambda: apply_rope_axes(t(1, 4, 8), t(4, 1, dtype=torch.int64), [(t(9, 5), t(9, 5))]), ValueError),
    (lambda: apply_rope_axes(t(1, 4, 8), t(4, 1, dtype=torch.int64), [(t(9, 2), t(9, 3))]), ValueError),
    (lambda: apply_rope_axes(t(1, 4, 8), t(4, 1, dtype=torch.int64), [(t(9), t(9))]), ValueError),
    (lambda: apply_rope_axes(t(1, 4, 8), t(5, 1, dtype=torch.int64), [(t(9, 2), t(9, 2))]), ValueError),
    (lambda: apply_rope_axes(t(2, 4, 8), t(3, 4, 1, dtype=torch.int64), [(t(9, 2), t(9, 2))]), ValueError),
    (lambda: apply_rope_axes(t(1, 4, 8), t(4, 1), [(t(9, 2), t(9, 2))]), TypeError),
    (lambda: apply_rope_axes(t(1, 4, 8), t(4, 1, dtype=torch.int64), [(t(9, 2), t(9, 2))]), RuntimeError),
])
def test_refusals(call, error):
    with pytest.raises(error):
        call()


def test_the_library_refuses_bad_arguments_before_it_launches():
    L = _abi.lib()
    n, m, r = _abi.LayerNormArgs(), _abi.LinearArgs(), _abi.RopeAxesArgs()
    assert L.pom_layer_norm_fwd(ctypes.byref(n), None) == -8
    n.x = n.y = 16
    assert L.pom_layer_norm_fwd(ctypes.byref(n), None) == -1  # no rows
    n.M, n.D, n.ldx, n.ldy = 2, 8, 7, 8
    assert L.pom_layer_norm_fwd(ctypes.byref(n), None) == -2
    n.ldx, n.bias = 8, 16
    assert L.pom_layer_norm_fwd(ctypes.byref(n), None) == -4  # a bias without a weight
    n.bias, n.dtype, n.wdtype = None, 1, 0
    assert L.pom_layer_norm_fwd(ctypes.byref(n), None) == -4  # bf16 weights beside float32 rows
    n.wdtype = 1
    assert L.pom_layer_norm_bwd(ctypes.byref(n), None) == -8  # no dy
    n.stats = 20
    assert L.pom_layer_norm_fwd(ctypes.byref(n), None) == -3
    assert L.pom_linear_fwd(ctypes.byref(m), None, None) == -1
    m.M, m.N, m.K = 4, 8, 8
    assert L.pom_linear_fwd(ctypes.byref(m), None, None) == -8
    m.x = m.w = m.y = 16
    m.ldx = m.ldw = 8
    assert L.pom_linear_fwd(ctypes.byref(m), None, None) == -2  # ldy
    m.ldy, m.act = 8, 9
    assert L.pom_linear_fwd(ctypes.byref(m), None, None) == -4
    m.act, m.dtype, m.M, m.K, m.ldx, m.ldw = 0, 1, 1000, 256, 256, 256
    assert L.pom_linear_fwd_workspace(ctypes.byref(m)) == 0  # a small product: the FMA kernel
    m.K = m.ldx = m.ldw = 1024
    assert L.pom_linear_fwd_workspace(ctypes.byref(m)) >= 6 * (1000 * 1024 + 8 * 1024)
    assert L.pom_linear_fwd(ctypes.byref(m), None, None) == -8  # float32 operands without room for their planes
    m.fma = 1
    assert L.pom_linear_fwd_workspace(ctypes.byref(m)) == 0
    m.fma = m.dtype = 0
    m.M, m.K, m.ldx, m.ldw = 4, 12, 12, 12
    assert L.pom_linear_fwd(ctypes.byref(m), None, None) == -2  # rows that bulk copies cannot address
    m.M, m.K, m.ldx, m.ldw, m.ld_dy, m.act = 64, 64, 64, 64, 8, 1
    assert L.pom_linear_bwd(ctypes.byref(m), None, None) == -8  # no dy
    m.dy = 16
    assert L.pom_linear_bwd(ctypes.byref(m), None, None) == -8  # an activation without its argument
    m.z = 16
    assert L.pom_linear_bwd_workspace(ctypes.byref(m)) >= 64 * 8 * 2
    assert L.pom_linear_bwd(ctypes.byref(m), None, None) == -8  # no workspace
    assert L.pom_rope_axes(ctypes.byref(r), None) == -8
    r.x = r.y = r.pos = 16
    assert L.pom_rope_axes(ctypes.byref(r), None) == -4
    r.axes, r.B, r.N, r.H, r.D = 1, 1, 1, 1, 8
    assert L.pom_rope_axes(ctypes.byref(r), None) == -8
    r.cos0 = r.sin0 = 16
    assert L.pom_rope_axes(ctypes.byref(r), None) == -1
    r.len0, r.pairs0 = 4, 5
    assert L.pom_rope_axes(ctypes.byref(r), None) == -1  # ten channels of eight
    assert L.pom_pos_range(None, 4, 1, None, None) == -8


def test_rows_of_takes_strides_as_they_are_or_copies():
    a = torch.arange(48.0).view(6, 8)
    assert ops.rows_of(a)[0] is a and ops.rows_of(a)[1] == 8
    b = a[:, :5]
    assert ops.rows_of(b)[0] is b and ops.rows_of(b)[1] == 8
    c = a.view(2, 3, 8)[:, :, 2:7]
    assert ops.rows_of(c)[0] is c and ops.rows_of(c)[1] == 8
    d = a.view(2, 3, 8)[:, :2]  # samples further apart than their rows
    got, ld = ops.rows_of(d)
    assert got.is_contiguous() and ld == 8 and torch.equal(got, d)
    for e in (a.t(), a[:1].expand(4, 8), a[:, :1].expand(6, 8)):
        got, ld = ops.rows_of(e)
        assert got.is_contiguous() and ld == e.shape[1] and torch.equal(got, e)
    one = a[2:3, 3:]  # a single row: the stride of a dimension of size 1 never matters
    assert ops.rows_of(one)[1] == 5
    shifted = torch.zeros(65, dtype=torch.bfloat16)[1:].view(8, 8)
    assert ops.rows_of(shifted)[0] is shifted
    assert ops.rows_of(shifted, align=True)[0].data_ptr() % 16 == 0


def test_tables_of_equal_axes_are_the_two_axis_tables():
    rc, rs, cc, cs = precompute_freqs_2d(64, 12, 9)
    (c0, s0), (c1, s1) = precompute_freqs_axes((16, 16), (12, 9))
    for got, want in ((c0, rc), (s0, rs), (c1, cc), (s1, cs)):
        assert got.shape == want.shape and got.dtype == torch.float32
        # the other tables form angles of up to 12 in float32: half a step of the frequency and of the product
        assert (got - want).abs().max() <= 12 * 3 * 2.0 ** -24
