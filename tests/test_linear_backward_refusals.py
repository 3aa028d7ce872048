"""The backward call of the linear operator at the C boundary: what bulk copies of bf16 rows cannot address is refused before
anything is launched.  No GPU."""
import ctypes

import pytest

from pom_b200 import _abi

STRIDE, ALIGN = -2, -3


def args(**kw):
    a = _abi.LinearArgs()
    base = dict(x=16, w=16, dy=16, z=16, workspace=256, M=64, N=64, K=64, ldx=64, ldw=64, ld_dy=64, act=1, dbias=16)
    for k, v in {**base, **kw}.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("kw, code", [
    (dict(N=65, ld_dy=72), STRIDE), (dict(ld_dy=68), STRIDE), (dict(dy=18), ALIGN), (dict(z=24), ALIGN),
    (dict(dx=8), ALIGN), (dict(dw=8), ALIGN), (dict(workspace=8), ALIGN), (dict(ld_dy=63), STRIDE)])
def test_bf16_rows_that_bulk_copies_cannot_address(kw, code):
    a = args(**kw)
    assert _abi.lib().pom_linear_bwd(ctypes.byref(a), None, None) == code


def test_the_backward_call_keeps_dz_in_its_workspace():
    assert not hasattr(_abi.LinearArgs(), "dz")
    a = args(dbias=None)
    assert _abi.lib().pom_linear_bwd_workspace(ctypes.byref(a)) == 64 * 64 * 2
