"""The linear operator keeps for its backward pass what that pass reads and no more: tokens under a frozen weight may change (or
go) once the product is done, and so may a weight whose tokens want no gradient."""
import pytest
import torch

from pom_b200.operators import linear

pytestmark = pytest.mark.gpu


def inputs(dtype, rows, wants):
    g = torch.Generator(device="cuda").manual_seed(3)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda").to(dtype)  # noqa: E731
    t = dict(x=r(rows, 72), w=r(40, 72), b=r(40), r=r(rows, 40))
    return {k: v.requires_grad_(k in wants) for k, v in t.items()}, r(rows, 40)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows", [5, 200])
@pytest.mark.parametrize("wants, frees", [("x", "x"), ("w", "w"), ("b", "xw"), ("r", "xw"), ("xb", "x"), ("wb", "w")])
@pytest.mark.parametrize("act", [None, "gelu"])
def test_what_is_not_read_again_may_change(act, wants, frees, rows, dtype):
    t, dy = inputs(dtype, rows, "xwbr")
    y = linear(t["x"], t["w"], t["b"], activation=act, residual=t["r"])
    want = dict(zip(wants, torch.autograd.grad(y, [t[k] for k in wants], dy)))
    t, dy = inputs(dtype, rows, wants)
    y = linear(t["x"], t["w"], t["b"], activation=act, residual=t["r"])
    with torch.no_grad():
        for k in frees:
            t[k].zero_()
    got = dict(zip(wants, torch.autograd.grad(y, [t[k] for k in wants], dy)))
    for k in wants:
        assert torch.equal(got[k], want[k]), k


def test_what_is_read_again_is_watched():
    for wants, changes in (("x", "w"), ("w", "x")):
        t, dy = inputs(torch.float32, 20, wants)
        y = linear(t["x"], t["w"])
        with torch.no_grad():
            t[changes].zero_()
        with pytest.raises(RuntimeError, match="inplace"):
            torch.autograd.grad(y, t[wants], dy)


def test_tokens_under_a_frozen_weight_are_let_go():
    w = torch.randn(1024, 1024, device="cuda", dtype=torch.bfloat16)
    x = torch.randn(16384, 1024, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    before = torch.cuda.memory_allocated()
    y = linear(x * 1, w)  # the product's input is an intermediate of 32 MB
    assert torch.cuda.memory_allocated() - before == y.numel() * 2


def test_padding_copies_only_what_has_the_odd_width():
    """An odd number of outputs pads the weight and the result, not the 32 MB of tokens; an odd sum pads no residual."""
    x = torch.randn(16384, 1024, device="cuda", dtype=torch.bfloat16)
    w = torch.randn(1001, 1024, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    y = linear(x, w)
    # the padded weight and result, and the result without its padding
    assert torch.cuda.max_memory_allocated() - before <= 2 * (1008 * 1024 + 16384 * 1008 + y.numel()) + (4 << 20)
    w = torch.randn(1024, 9, device="cuda", dtype=torch.bfloat16)
    r = torch.randn(16384, 1024, device="cuda", dtype=torch.bfloat16)
    x = torch.randn(16384, 9, device="cuda", dtype=torch.bfloat16)
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    y = linear(x, w, residual=r)
    assert torch.cuda.max_memory_allocated() - before <= 2 * (16384 * 16 + 1024 * 16 + y.numel()) + (4 << 20)
