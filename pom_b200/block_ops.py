"""Operators of a residual block around the mixer, on the CUDA kernels of this package: layer norm, the linear map with
bias, activation and residual, and rotary positions of several axes.

The reference leaves the first two to ``torch.nn`` and has rotary positions of one and two axes
(pom/pom_rope.py:152-235).  All three take bfloat16 and float32 tensors, any strides (rows that do not follow one another
in one step are copied), run on the tensors' device and current stream, are differentiable once (backward; a forward-mode
tangent is refused), and may be captured into CUDA graphs.  They give the same bits on every run.  ``pom_b200.operators``
exports them.

A backward pass is captured together with its forward pass, and, as with PyTorch's own operators, while no eager graph of
the same leaves is alive (autograd would join the capture with the stream that such a graph was made on; it raises).
"""
from __future__ import annotations

import functools
from typing import Optional, Sequence, Tuple

import torch
import torch.nn.functional as F
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _abi, ops
from .functional import eager_only

_any_autocast = getattr(torch._C, "_is_any_autocast_enabled", lambda: True)
_TYPES = (torch.bfloat16, torch.float32)


def _check_tokens(x: torch.Tensor, name: str = "x") -> None:
    # where it lives is checked with the other tensors of the call (ops._same_device)
    if not isinstance(x, torch.Tensor):
        raise TypeError(f"{name} must be a tensor, got {type(x).__name__}")
    if x.dtype not in _TYPES:
        raise TypeError(f"unsupported dtype {x.dtype} of {name}; use bfloat16 or float32")


_current_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device


def _has_tangent(t) -> bool:
    if isinstance(t, torch.Tensor):
        return forward_ad.unpack_dual(t).tangent is not None
    return isinstance(t, (tuple, list)) and any(_has_tangent(e) for e in t)


def _entry(fn):
    """``eager_only``, a refusal of forward-mode derivatives (untracked calls do not go through autograd, which would refuse
    them), and a switch to the device of the first argument, as the package's other entry points make it; one wrapper of
    few steps, because a small call costs the host more than the GPU."""

    @eager_only
    @functools.wraps(fn)
    def wrapper(x, *args, **kwargs):
        if getattr(forward_ad, "_current_level", 0) >= 0 and _has_tangent((x, *args, *kwargs.values())):
            raise NotImplementedError(f"{fn.__name__} has no forward-mode derivative: differentiate it backward")
        if isinstance(x, torch.Tensor):
            i = x.get_device()
            if i >= 0 and i != _current_device():
                with torch.cuda.device(i):
                    return fn(x, *args, **kwargs)
        return fn(x, *args, **kwargs)

    return wrapper


def _backward(fn):
    """A backward pass that is differentiable once.  Under ``create_graph`` it goes through ``once_differentiable``, whose
    outputs refuse a second differentiation; the ordinary case does without that wrapper.  The engine calls it with the
    device of the forward call current."""
    checked = once_differentiable(fn)

    @functools.wraps(fn)
    def wrapper(ctx, g):
        return checked(ctx, g) if torch.is_grad_enabled() else fn(ctx, g)

    return staticmethod(wrapper)


# --------------------------------------------------------------------------- layer norm
class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        y, stats = ops.layer_norm_fwd(x, weight, bias, eps, True)
        ctx.save_for_backward(x, weight, stats)
        return y

    @_backward
    def backward(ctx, g):
        x, weight, stats = ctx.saved_tensors
        nx, nw, nb, _ = ctx.needs_input_grad
        dx, dw, db = ops.layer_norm_bwd(g, x, weight, stats, want_dx=nx, want_dw=nw, want_db=nb)
        return dx, dw, db, None


@_entry
def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
               eps: float = 1e-5) -> torch.Tensor:
    """``(x - mean) / sqrt(var + eps) * weight + bias`` over the last dimension, in x's dtype.

    x (..., D) bfloat16 or float32; ``weight`` and ``bias`` (D,) in x's dtype or float32 (``bias`` only with ``weight``).
    Statistics and sums are float32, so a row's sum and its sum of squared deviations must stay below 3e38 (values up to
    1e15 always do).  A row with an infinity or a NaN comes out NaN."""
    _check_tokens(x)
    if x.dim() < 1 or x.shape[-1] == 0:
        raise ValueError(f"expected a (..., D) tensor with D > 0, got {tuple(x.shape)}")
    if weight is None:
        if bias is not None:
            raise ValueError("layer_norm takes a bias only together with a weight")
    else:
        D = x.shape[-1]
        for t, name in ((weight, "weight"), (bias, "bias")):
            if t is None:
                continue
            _check_tokens(t, name)
            if t.dim() != 1 or t.shape[0] != D:
                raise ValueError(f"{name} must have shape ({D},), got {tuple(t.shape)}")
        if weight.dtype != torch.float32 and weight.dtype != x.dtype:
            weight = weight.float()  # bf16 parameters beside float32 rows
        if not weight.is_contiguous():
            weight = weight.contiguous()
        if bias is not None:
            if bias.dtype != weight.dtype:
                if weight.dtype == torch.bfloat16:
                    weight = weight.float()
                bias = bias.to(weight.dtype)
            if not bias.is_contiguous():
                bias = bias.contiguous()
    if torch.is_grad_enabled() and (x.requires_grad or (weight is not None and weight.requires_grad) or
                                    (bias is not None and bias.requires_grad)):
        return _LayerNorm.apply(x, weight, bias, eps)
    return ops.layer_norm_fwd(x, weight, bias, eps, False)[0]


# --------------------------------------------------------------------------- linear map
class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, act):
        nx, nw, nb, _, _ = ctx.needs_input_grad
        y, z = ops.linear_fwd(x, weight, bias, act, residual, act is not None and (nx or nw or nb))
        ctx.save_for_backward(x if nw else None, weight if nx else None, z)
        ctx.act = act
        ctx.bias_dtype = bias.dtype if nb else None
        return y

    @_backward
    def backward(ctx, g):
        x, weight, z = ctx.saved_tensors
        nx, nw, nb, nr, _ = ctx.needs_input_grad
        dx = dw = db = None
        if nx or nw or nb:
            dx, dw, db = ops.linear_bwd(g, x, weight, ctx.act, z, want_dx=nx, want_dw=nw, bias_dtype=ctx.bias_dtype)
        return dx, dw, db, (g if nr else None), None


def _pad8(n: int) -> int:
    return -n % 8


def _padded(t: Optional[torch.Tensor], *pad: int) -> Optional[torch.Tensor]:
    return t if t is None or not any(pad) else F.pad(t, pad)  # (padding by nothing would copy)


@_entry
def linear(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, *,
           activation: Optional[str] = None, residual: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``activation(x · weightᵀ + bias) + residual`` in one product.

    x (..., K) and ``weight`` (N, K) of one dtype, bfloat16 or float32; ``bias`` (N,) in that dtype or float32;
    ``residual`` of the output's shape and dtype; ``activation`` None, "gelu" (exact), "gelu_tanh", "silu" or "relu".
    Sums, bias, activation and residual are float32, rounded once.  Under ``torch.autocast("cuda", torch.bfloat16)`` x,
    ``weight`` and ``residual`` are cast to bfloat16 on the way in, and y is bfloat16.

    Gradients: with an activation its argument z is kept in x's dtype, and dz, what comes back through the activation, is
    rounded to it before dW = dzᵀ x and dx = dz W.  In bfloat16 those two carry two roundings instead of one (0.0024 of
    their norm against 0.0017); without an activation dz is the incoming gradient, and nothing is added.

    bfloat16 widths that are not multiples of 8 are padded with zeros (a copy of the operands that have them), but for N
    of up to 16 (K up to 2048: 32) rows without a gradient.  float32 products take a workspace of three bfloat16 planes per operand; where
    memory has no room for it, they run as chains of fused multiply-adds over the whole sum, whose error grows with K."""
    _check_tokens(x)
    _check_tokens(weight, "weight")
    if activation not in _abi.ACTIVATIONS:
        raise ValueError(f"activation must be one of {sorted(k for k in _abi.ACTIVATIONS if k)} or None, got {activation!r}")
    if weight.dim() != 2 or x.dim() < 1 or x.shape[-1] != weight.shape[1] or 0 in weight.shape:
        raise ValueError(f"expected x (..., K) and weight (N, K) with N, K > 0, got {tuple(x.shape)} and {tuple(weight.shape)}")
    N, K = weight.shape
    if bias is not None:
        _check_tokens(bias, "bias")
        if bias.shape != (N,):
            raise ValueError(f"bias must have shape ({N},), got {tuple(bias.shape)}")
    if residual is not None:
        _check_tokens(residual, "residual")
        if residual.shape[:-1] != x.shape[:-1] or residual.shape[-1] != N:
            raise ValueError(f"residual must have the output's shape {(*x.shape[:-1], N)}, got {tuple(residual.shape)}")
    if _any_autocast():
        from .pom import PoM  # the module decides what autocast means for its projections; the same here

        dt = PoM._autocast_dtype()
        if dt is not None:
            x, weight = x.to(dt), weight.to(dt)
            residual = None if residual is None else residual.to(dt)
    if weight.dtype != x.dtype or (residual is not None and residual.dtype != x.dtype):
        raise TypeError("x, weight and residual must share one dtype")
    if bias is not None:
        if x.dtype == torch.float32 and bias.dtype != torch.float32:
            bias = bias.float()
        bias = bias.contiguous()
    tracked = torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad or (bias is not None and bias.requires_grad)
                                           or (residual is not None and residual.requires_grad))
    # the kernel for few rows takes any N; bulk copies and the backward pass do not
    if x.dtype == torch.bfloat16 and (K % 8 or (N % 8 and (tracked or x.numel() > _abi.linear_few_rows(K) * K))):
        kp, n_pad = _pad8(K), _pad8(N)
        y = linear(_padded(x, 0, kp), _padded(weight, 0, kp, 0, n_pad), _padded(bias, 0, n_pad), activation=activation,
                   residual=_padded(residual, 0, n_pad))
        return y[..., :N].contiguous() if n_pad else y
    if tracked:
        return _Linear.apply(x, weight, bias, residual, activation)
    return ops.linear_fwd(x, weight, bias, activation, residual, False)[0]


# --------------------------------------------------------------------------- rotary positions of several axes
class _RotateAxes(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, pos, tables):
        ctx.save_for_backward(pos, *(t for pair in tables for t in pair))  # an update in place before backward is noticed
        return ops.rope_axes(x, pos, tables)

    @_backward
    def backward(ctx, g):
        pos, *flat = ctx.saved_tensors
        return ops.rope_axes(g, pos, list(zip(flat[::2], flat[1::2])), transpose=True), None, None


def _f32_on(t: torch.Tensor, device: int, x: torch.Tensor) -> torch.Tensor:
    if t.dtype == torch.float32 and t.get_device() == device and t.is_contiguous():
        return t
    return t.to(device=x.device, dtype=torch.float32).contiguous()


@_entry
def apply_rope_axes(x: torch.Tensor, positions: torch.Tensor, tables: Sequence[Tuple[torch.Tensor, torch.Tensor]], *,
                    validate: bool = True) -> torch.Tensor:
    """Rotary positions of one to four axes, e.g. (time, height, width) of video tokens.

    x (B, N, D), or (B, N, H, D) with heads that share the angles.  ``tables``: per axis a (cos, sin) pair of
    (rows, s_a) tensors (see :func:`precompute_freqs_axes`); the axes' sections of 2 s_a channels follow one another, and
    inside a section channel k pairs with k + s_a, as :func:`apply_rope_2d` pairs its two halves; channels behind the
    last section pass.  ``positions`` (N, A) for all samples, or (B, N, A).  Only x has a gradient.  Tables and positions
    of another device or type are copied in every call.

    ``validate``: an IndexError for a position outside its table, for which the call waits until the stream has come
    to it (and cannot be captured).  Without it nothing is read back, and such a position makes its section of the token
    NaN.  Nothing is remembered between calls: a model that rotates by the same positions in every layer checks them in
    its first call and passes ``validate=False`` in the others, so that only one call waits."""
    _check_tokens(x)
    if x.dim() not in (3, 4):
        raise ValueError(f"expected a (B, N, D) or (B, N, H, D) tensor, got {tuple(x.shape)}")
    if not 1 <= len(tables) <= _abi.ROPE_MAX_AXES:
        raise ValueError(f"1 to {_abi.ROPE_MAX_AXES} axes, got {len(tables)}")
    D, axes, width, tabs = x.shape[-1], len(tables), 0, []
    device = x.get_device()
    for cos, sin in tables:
        shape = cos.shape
        if len(shape) != 2 or shape != sin.shape or 0 in shape:
            raise ValueError(f"every table must be two (rows, pairs) tensors of one shape, got {tuple(shape)} and "
                             f"{tuple(sin.shape)}")
        if (cos.requires_grad or sin.requires_grad) and torch.is_grad_enabled():
            raise ValueError("the tables take no gradient: pass them detached")
        width += 2 * shape[1]
        tabs.append((_f32_on(cos, device, x), _f32_on(sin, device, x)))
    if width > D:
        raise ValueError(f"the axes rotate {width} channels but x has {D}")
    B, N = x.shape[:2]
    if positions.shape != (N, axes) and positions.shape != (B, N, axes):
        raise ValueError(f"positions must have shape ({N}, {axes}) or ({B}, {N}, {axes}), got {tuple(positions.shape)}")
    pos = positions
    if pos.dtype != torch.int64 or pos.get_device() != device:
        if pos.dtype.is_floating_point or pos.dtype == torch.bool or pos.dtype.is_complex:
            raise TypeError(f"positions must be integers, got {pos.dtype}")
        pos = pos.to(device=x.device, dtype=torch.int64)
    if not pos.is_contiguous():
        pos = pos.contiguous()
    validate = validate and pos.numel() > 0
    # the rotation follows at once (a bad position is harmless there); only the answer is waited for
    started = ops.pos_range_start(pos) if validate else None
    found = ()
    try:
        y = _RotateAxes.apply(x, pos, tabs) if x.requires_grad and torch.is_grad_enabled() else ops.rope_axes(x, pos, tabs)
    finally:
        if started is not None:
            found = ops.pos_range_wait(started)
    for a, ((lo, hi), (cos, _)) in enumerate(zip(found, tabs)):
        if lo < 0 or hi >= cos.shape[0]:
            raise IndexError(f"positions of axis {a} span [{lo}, {hi}] but its table has {cos.shape[0]} rows")
    return y


def precompute_freqs_axes(pairs: Sequence[int], rows: Sequence[int], base: float = 10000.0, *, device=None):
    """One (cos, sin) pair of (rows[a], pairs[a]) float32 tables per axis, angle position * base^(-k / pairs[a]); formed in
    64 bits, so that far positions keep their angles.  They are wanted on the ``device`` of the tokens: made once, there.
    With equal axes the tables of :func:`pom_b200.pom_rope.precompute_freqs_2d`."""
    out = []
    for s, n in zip(pairs, rows):
        f = float(base) ** (-torch.arange(s, dtype=torch.float64) / s)
        ang = torch.outer(torch.arange(n, dtype=torch.float64), f)
        out.append((ang.cos().float().to(device), ang.sin().float().to(device)))
    return out
