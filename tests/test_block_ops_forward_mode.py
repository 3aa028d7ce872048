"""Forward-mode derivatives of layer norm, linear and several-axis rotary operators are refused, whichever argument carries the
tangent and however it is passed; nothing is computed without it.  No GPU: the refusal comes before the device is looked at."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

from pom_b200 import ops
from pom_b200.operators import apply_rope_axes, layer_norm, linear


@pytest.fixture(autouse=True)
def no_kernels(monkeypatch):
    """What an untracked call launches, as elementary operations without derivatives."""
    monkeypatch.setattr(ops, "layer_norm_fwd", lambda x, *a: (x.detach().clone(), None))
    monkeypatch.setattr(ops, "linear_fwd", lambda x, w, *a: ((x @ w.t()).detach(), None))
    monkeypatch.setattr(ops, "rope_axes", lambda x, *a: x.detach().clone())


def t(*shape):
    return torch.ones(*shape)


CALLS = [
    (layer_norm, dict(x=t(2, 8), weight=t(8), bias=t(8)), ("x", "weight", "bias")),
    (linear, dict(x=t(2, 8), weight=t(4, 8), bias=t(4), residual=t(2, 4)), ("x", "weight", "bias", "residual")),
    (apply_rope_axes, dict(x=t(1, 2, 8), positions=torch.zeros(2, 1, dtype=torch.int64), tables=[(t(3, 2), t(3, 2))],
                           validate=False), ("x",)),
]


@pytest.mark.parametrize("fn, kwargs, name", [(fn, kw, n) for fn, kw, names in CALLS for n in names])
def test_a_tangent_is_refused(fn, kwargs, name):
    with fwd.dual_level():
        dual = fwd.make_dual(kwargs[name], torch.ones_like(kwargs[name]))
        rest = {k: v for k, v in kwargs.items() if k not in ("x", name)}
        for call in (lambda: fn(**{**kwargs, name: dual}),
                     lambda: fn(dual if name == "x" else kwargs["x"], **rest, **({} if name == "x" else {name: dual}))):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call()
        with torch.no_grad(), pytest.raises(NotImplementedError, match="forward-mode"):
            fn(**{**kwargs, name: dual})


def test_a_tangent_of_a_table_is_refused():
    fn, kwargs, _ = CALLS[2]
    for which in (0, 1):
        with fwd.dual_level():
            pair = [t(3, 2), t(3, 2)]
            pair[which] = fwd.make_dual(pair[which], t(3, 2))
            with pytest.raises(NotImplementedError, match="forward-mode"):
                fn(**{**kwargs, "tables": [tuple(pair)]})


@pytest.mark.parametrize("fn, kwargs, names", CALLS)
def test_calls_without_a_tangent_run_inside_a_dual_level(fn, kwargs, names):
    with fwd.dual_level():
        fwd.make_dual(t(2), t(2))  # somebody else's
        fn(**kwargs)
    fn(**kwargs)


def test_jvp_of_torch_func_is_refused():
    with pytest.raises(Exception):
        torch.func.jvp(lambda x: layer_norm(x), (t(2, 8),), (t(2, 8),))
