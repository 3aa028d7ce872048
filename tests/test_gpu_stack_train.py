"""PoMStack with norms, biases and a backward pass: layer norm, mixer and feed-forward products in a row, against the CPU
oracle's mixer and torch's elementary operators in float64."""
import pytest
import torch

from oracle import pom_oracle as O
from pom_b200 import BlockCausal
from pom_b200.stack import PoMStack
from tests.helpers import BF16_TOL, FP32_TOL

pytestmark = pytest.mark.gpu

ACTS = {"gelu": torch.nn.functional.gelu, "gelu_tanh": lambda z: torch.nn.functional.gelu(z, approximate="tanh"),
        "silu": torch.nn.functional.silu, "relu": torch.relu}


def make(D, layers, dtype, seed=5, **kw):
    torch.manual_seed(seed)
    stack = PoMStack(D, 2, 2, layers, **kw)
    with torch.no_grad():
        for m in stack.mixers:
            m.po_coeff.copy_(torch.randn_like(m.po_coeff) * 0.1)
        for m in [*stack.norm_mix, *stack.norm_ffn]:
            m.weight.add_(torch.randn_like(m.weight) * 0.2)
            m.bias.add_(torch.randn_like(m.bias) * 0.2)
        for p in stack.parameters():
            p.copy_(O.bf16_round(p))
    params = {k: v.detach().clone() for k, v in stack.named_parameters()}
    return stack.cuda().to(dtype), params


def reference(params, stack, x, mask):
    """The stack's definition on the oracle's mixer, from a dict of float64 parameters."""
    h = x
    for i in range(len(stack.mixers)):
        own = {k.split(".", 2)[2]: v for k, v in params.items() if k.startswith(f"mixers.{i}.")}
        mixer = O.OraclePoM(own, 2, 2)

        def normed(name, t):
            if f"{name}.{i}.weight" not in params:
                return t
            return torch.nn.functional.layer_norm(t, t.shape[-1:], params[f"{name}.{i}.weight"], params[f"{name}.{i}.bias"])

        h = h + mixer.forward(normed("norm_mix", h), mask=mask)
        u = normed("norm_ffn", h) @ params[f"ffn_in.{i}.weight"].t()
        if f"ffn_in.{i}.bias" in params:
            u = u + params[f"ffn_in.{i}.bias"]
        u = ACTS[stack.activation](u) @ params[f"ffn_out.{i}.weight"].t()
        if f"ffn_out.{i}.bias" in params:
            u = u + params[f"ffn_out.{i}.bias"]
        h = h + u
    return h


def rel(a, b):
    return ((a.double().cpu() - b).norm() / b.norm().clamp_min(1e-30)).item()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("mask, kw", [
    (None, dict(norm=True, bias=True)), ("causal", dict(norm=True, bias=True, activation="silu")),
    ("pad", dict(norm=True, activation="gelu_tanh")), ("block", dict(norm=True, bias=True, activation="relu")),
    (None, dict()), ("causal", dict(bias=True))])
def test_stack_gradients(mask, kw, dtype):
    if mask == "block" and dtype == torch.float32:
        mask = "causal"  # block-causal masks are a bfloat16 path
    B, N, D, layers = 2, 96, 64, 2
    stack, params = make(D, layers, dtype, **kw)
    x, gy = O.bf16_round(torch.randn(B, N, D)), O.bf16_round(torch.randn(B, N, D))
    m_ref = m_own = mask
    if mask == "pad":
        m_ref = (torch.arange(N)[None] < torch.tensor([[N], [41]])).double()
        m_own = m_ref.float().cuda()
    elif mask == "block":
        m_ref, m_own = O.block_causal_mask(N, 32, B, dtype=torch.float64), BlockCausal(32)
    ps = {k: v.double().requires_grad_(True) for k, v in params.items()}
    xr = x.double().requires_grad_(True)
    want = reference(ps, stack, xr, m_ref)
    want_g = torch.autograd.grad(want, [xr, *ps.values()], gy.double())
    xg = x.cuda().to(dtype).requires_grad_(True)
    y = stack.train_forward(xg, m_own)
    named = dict(stack.named_parameters())
    got_g = torch.autograd.grad(y, [xg, *[named[k] for k in ps]], gy.cuda().to(dtype))
    # the bounds that the mixer's own tests allow one layer, for two layers and their feed-forward blocks
    tol = 3 * BF16_TOL if dtype == torch.bfloat16 else 4 * FP32_TOL
    assert rel(y, want) <= tol
    if dtype == torch.bfloat16 and stack.activation == "relu":
        # relu's slope jumps at 0.  About ten stored bf16 values stand before a pre-activation z (tokens, norms, the mixer's
        # projections, gate and output), each off by 2^-9 / sqrt 3 of itself: d = 10^(1/2) * 1.1e-3 = 3.6e-3 of z's spread.
        # A normal z lies within its error of 0 with probability 2 * 0.4 * 0.8 d = 2.3e-3, and then the slope, hence that
        # element of dz, is wrong by all of it; half of the elements have slope 1, so dz is off by (2 * 2.3e-3)^(1/2) =
        # 6.8e-2 in the 2-norm per layer, and so is what is summed from it
        tol = (tol ** 2 + layers * 6.8e-2 ** 2) ** 0.5
    for name, a, b in zip(["x", *ps], got_g, want_g):
        assert a.dtype == dtype
        assert rel(a, b) <= tol, (name, rel(a, b))


def test_inference_paths_agree_with_the_training_path():
    B, F, L, D = 2, 4, 64, 64
    for kw in (dict(norm=True, bias=True, activation="silu"), dict(norm=True), dict(bias=True), dict()):
        stack, params = make(D, 3, torch.bfloat16, **kw)
        x = O.bf16_round(torch.randn(B, F * L, D))
        want = reference({k: v.double() for k, v in params.items()}, stack, x.double(),
                         O.block_causal_mask(F * L, L, B, dtype=torch.float64))
        xg = x.cuda().bfloat16()
        loop, one = stack(xg, L), stack.forward_single_pass(xg, L)
        with torch.no_grad():
            train = stack.train_forward(xg, BlockCausal(L))
        for got in (loop, one, train):
            assert rel(got, want) <= 3 * BF16_TOL


def test_autocast_and_a_training_step():
    stack, params = make(64, 2, torch.float32, norm=True, bias=True)
    x = O.bf16_round(torch.randn(2, 96, 64)).cuda()
    opt = torch.optim.SGD(stack.parameters(), lr=1e-3)
    before = {k: v.detach().clone() for k, v in stack.named_parameters()}
    with torch.autocast("cuda", torch.bfloat16):
        loss = stack.train_forward(x, "causal").float().square().mean()
    loss.backward()
    ps = {k: v.double().requires_grad_(True) for k, v in params.items()}
    want = torch.autograd.grad(reference(ps, stack, x.double().cpu(), "causal").square().mean(), list(ps.values()))
    for (k, p), g in zip(stack.named_parameters(), want):
        assert p.grad.dtype == torch.float32 and rel(p.grad, g) <= 3 * BF16_TOL, k
    opt.step()
    assert all(not torch.equal(before[k], v) for k, v in stack.named_parameters())


def test_captured_training_step():
    stack, _ = make(64, 2, torch.bfloat16, norm=True, bias=True)
    x, gy = torch.randn(2, 96, 64, device="cuda").bfloat16(), torch.randn(2, 96, 64, device="cuda").bfloat16()
    ps = list(stack.parameters())

    def step():
        return torch.autograd.grad(stack.train_forward(x, "causal"), ps, gy)

    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = step()
    for _ in range(2):
        g.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert rel(a, b.double().cpu()) <= 1e-2  # the mixer's own weight gradients are summed by atomics
            a.zero_()


def test_default_stack_keeps_its_parameters():
    torch.manual_seed(3)
    a = PoMStack(64, 2, 2, 2)
    assert not any("norm" in k or k.startswith("ffn") and k.endswith("bias") for k in a.state_dict())
    with pytest.raises(ValueError):
        PoMStack(64, 2, 2, 1, activation="tanh")
    with pytest.raises(TypeError):
        a.train_forward(torch.zeros(1, 8, 64))
