"""The block operators whose speed is followed: layer norm, the linear map with bias, activation and residual, and rotary
positions of several axes, each with the elementary torch form of the same arithmetic (``own`` false) beside the
framework's call (``own`` true) and its definition in 64 bits (``exact``).

A case is a dict of plain values:

* ``op``     "norm" | "linear" | "rope"
* ``family`` what the case stands for; :func:`draw` varies the sizes inside a family
* ``dtype``  "bf16" | "fp32" of the tokens; ``train``: with the gradients of every floating input
* norm:   ``M`` rows, ``D`` channels, ``affine``, ``wdtype`` of the scale and the shift
* linear: ``M`` rows, ``K`` -> ``N`` channels, ``bias``, ``act`` "none" | "gelu" | "gelu_tanh" | "silu" | "relu", ``res``
* rope:   ``B`` samples, ``T`` x ``Y`` x ``X`` grid, ``H`` heads (0: none), ``D`` channels, ``st, sy, sx`` pairs per axis,
          ``own_pos`` one position list per sample, ``checked`` positions compared with the tables before the launch
"""
import math

import torch

own = False

_NORM = dict(op="norm", dtype="bf16", train=True, affine=True, wdtype="bf16")
_LINEAR = dict(op="linear", dtype="bf16", train=True, bias=True, act="none", res=False)
_ROPE = dict(op="rope", dtype="bf16", train=True, H=0, own_pos=False, checked=True)


def listed():
    return [
        # One token of eight videos, before the mixer of a stack that answers token by token: the smallest call.
        dict(_NORM, name="norm_token", family="norm_token", train=False, M=8, D=1024),
        # A training step of the image-generation layer: 32 images of 32 x 32 patches.
        dict(_NORM, name="norm_train", family="norm_train", M=32768, D=1152),
        # One long sequence, its scale and shift kept in float32.
        dict(_NORM, name="norm_long", family="norm_train", M=65536, D=1152, wdtype="fp32"),
        # A float32 experiment, an odd number of rows.
        dict(_NORM, name="norm_fp32", family="norm_fp32", dtype="fp32", wdtype="fp32", M=4079, D=1152),
        # First feed-forward product for one token of eight videos: the weight is what is read.
        dict(_LINEAR, name="linear_token", family="linear_token", train=False, M=8, K=1024, N=4096, act="gelu"),
        # Second feed-forward product of one 256-token frame of eight videos.
        dict(_LINEAR, name="linear_frame", family="linear_frame", train=False, M=2048, K=4096, N=1024, res=True),
        # Both feed-forward products of the image-generation layer in training: the largest calls.
        dict(_LINEAR, name="linear_up_train", family="linear_train", M=32768, K=1152, N=4608, act="gelu"),
        dict(_LINEAR, name="linear_down_train", family="linear_train", M=32768, K=4608, N=1152, res=True),
        # A float32 experiment.
        dict(_LINEAR, name="linear_fp32_train", family="linear_fp32", dtype="fp32", M=4079, K=384, N=1536, act="silu"),
        # Features of a video of 16 frames of 32 x 32 patches, two samples on one grid.
        dict(_ROPE, name="rope_video_train", family="rope_train", B=2, T=16, Y=32, X=32, D=2304, st=384, sy=384, sx=384),
        # Videos of different places in one batch, several heads, channels that no axis rotates.
        dict(_ROPE, name="rope_heads_train", family="rope_heads", B=6, T=5, Y=15, X=20, H=16, D=72, st=8, sy=12, sx=12,
             own_pos=True),
        # The next token of eight videos, each at its own position.
        dict(_ROPE, name="rope_token", family="rope_token", train=False, B=8, T=1, Y=1, X=1, D=2304, st=384, sy=384,
             sx=384, own_pos=True, checked=False),
    ]


# ---------------------------------------------------------------------------- drawn cases
def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi, odd):
    """Channels: multiples of 8 as a rule, any number one time in ``odd``."""
    w = _log_int(rng, lo, hi)
    return w if rng.randrange(odd) == 0 else max(8, w // 8 * 8)


def draw(rng):
    family = rng.choice(["norm_token", "norm_train", "norm_fp32", "linear_token", "linear_frame", "linear_train",
                         "linear_fp32", "rope_train", "rope_heads", "rope_token"])
    act = rng.choice(["none", "gelu", "gelu_tanh", "silu", "relu"])
    flags = dict(bias=rng.random() < 0.8, act=act, res=rng.random() < 0.5)
    if family == "norm_token":
        return dict(_NORM, family=family, train=False, M=_log_int(rng, 1, 256), D=_width(rng, 64, 4608, 4))
    if family == "norm_train":
        D = _width(rng, 128, 4608, 5)
        return dict(_NORM, family=family, D=D, M=_log_int(rng, 256, 37_000_000 // D), affine=rng.random() < 0.8,
                    wdtype=rng.choice(["bf16", "fp32"]))
    if family == "norm_fp32":
        D = _width(rng, 96, 2304, 4)
        return dict(_NORM, family=family, dtype="fp32", wdtype="fp32", D=D, M=_log_int(rng, 64, 9_000_000 // D))
    if family == "linear_token":
        return dict(_LINEAR, family=family, train=False, M=_log_int(rng, 1, 64), K=_width(rng, 128, 4608, 8),
                    N=_width(rng, 128, 4608, 8), **flags)
    if family in ("linear_frame", "linear_train"):
        K, N = _width(rng, 256, 4608, 8), _width(rng, 256, 4608, 8)
        most = 32768 * 1152 * 4608 // (K * N)
        train = family == "linear_train"
        M = _log_int(rng, 512 if train else 65, min(most, 32768 if train else 4096))
        return dict(_LINEAR, family=family, train=train, M=M, K=K, N=N, **flags)
    if family == "linear_fp32":
        return dict(_LINEAR, family=family, dtype="fp32", M=_log_int(rng, 1, 4096), K=_width(rng, 64, 1536, 4),
                    N=_width(rng, 64, 1536, 4), train=rng.random() < 0.7, **flags)
    if family == "rope_token":
        s = [rng.randint(16, 400) for _ in range(3)]
        return dict(_ROPE, family=family, train=False, B=_log_int(rng, 1, 64), T=1, Y=1, X=1, own_pos=True, checked=False,
                    D=2 * sum(s) + rng.choice([0, 0, 8, 64]), **dict(zip(("st", "sy", "sx"), s)))
    T, Y, X = rng.randint(1, 16), rng.randint(4, 40), rng.randint(4, 40)
    heads = family == "rope_heads"
    step = rng.choice([1, 4, 8, 8])
    s = [step * rng.randint(1, (48 if heads else 400) // step) for _ in range(3)]
    D = 2 * sum(s) + rng.choice([0, 0, 16])
    H = rng.randint(2, 16) if heads else 0
    B = _log_int(rng, 1, max(1, min(64, 36_000_000 // (T * Y * X * D * max(H, 1)))))
    return dict(_ROPE, family=family, B=B, T=T, Y=Y, X=X, H=H, D=D, dtype=rng.choice(["bf16", "bf16", "fp32"]),
                own_pos=heads and rng.random() < 0.5, **dict(zip(("st", "sy", "sx"), s)))


# ---------------------------------------------------------------------------- inputs
_TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
_LEN = 512  # rows of the rotary tables


def _table(pairs):
    """cos and sin of position * 10000^(-k / pairs), angles in 64 bits."""
    f = 10000.0 ** (-torch.arange(pairs, dtype=torch.float64, device="cuda") / pairs)
    a = torch.arange(_LEN, dtype=torch.float64, device="cuda")[:, None] * f
    return a.cos().float(), a.sin().float()


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt, train = _TYPES[case["dtype"]], case["train"]

    def normal(*shape, scale=1.0, dtype=dt, leaf=True):
        t = torch.randn(*shape, generator=g, device="cuda").mul_(scale).to(dtype)
        return t.requires_grad_(train and leaf)

    s = dict(case=case)
    if case["op"] == "norm":
        M, D, wdt = case["M"], case["D"], _TYPES[case["wdtype"]]
        # a residual stream: channels of different sizes around different means, rows of different sizes
        x = torch.randn(M, D, generator=g, device="cuda")
        x *= torch.rand(D, generator=g, device="cuda").mul_(3).add_(0.3)
        x += torch.randn(D, generator=g, device="cuda").mul_(0.7)
        x *= torch.rand(M, 1, generator=g, device="cuda").mul_(2).add_(0.2)
        s["x"] = x.to(dt).requires_grad_(train)
        if case["affine"]:
            s["w"] = torch.randn(D, generator=g, device="cuda").mul_(0.2).add_(1).to(wdt).requires_grad_(train)
            s["b"] = normal(D, scale=0.1, dtype=wdt)
        s["dy"] = normal(M, D, leaf=False) if train else None
    elif case["op"] == "linear":
        M, N, K = case["M"], case["N"], case["K"]
        s["x"] = normal(M, K)
        s["w"] = normal(N, K, scale=K ** -0.5)
        s["b"] = normal(N, scale=0.2) if case["bias"] else None
        s["r"] = normal(M, N) if case["res"] else None
        s["dy"] = normal(M, N, leaf=False) if train else None
    else:
        B, T, Y, X = case["B"], case["T"], case["Y"], case["X"]
        n = T * Y * X
        heads = (case["H"],) if case["H"] else ()
        s["x"] = normal(B, n, *heads, case["D"])
        i = torch.arange(n, device="cuda")
        pos = torch.stack([i // (Y * X), i // X % Y, i % X], -1)
        if case["own_pos"]:  # each sample begins somewhere else
            pos = pos + torch.randint(0, _LEN - 64, (B, 1, 3), generator=g, device="cuda")
        s["pos"] = pos
        s["tables"] = [_table(case[k]) for k in ("st", "sy", "sx")]
        s["dy"] = normal(B, n, *heads, case["D"], leaf=False) if train else None
    return s


def _leaves(s):
    return [s[k] for k in ("x", "w", "b", "r") if s.get(k) is not None]


# ---------------------------------------------------------------------------- plain forms
_C = math.sqrt(2 / math.pi)


def _act(z, kind):
    """act(z) and act'(z)."""
    if kind == "relu":
        return z.clamp(min=0), (z > 0).to(z.dtype)
    if kind == "silu":
        p = 1 / (1 + torch.exp(-z))
        return z * p, p * (1 + z * (1 - p))
    if kind == "gelu":
        c = 0.5 * (1 + torch.erf(z * math.sqrt(0.5)))
        return z * c, c + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    t = torch.tanh(_C * (z + 0.044715 * z * z * z))
    return 0.5 * z * (1 + t), 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * _C * (1 + 3 * 0.044715 * z * z)


def _plain_norm(s):
    c, x = s["case"], s["x"].float()
    w = s["w"].float() if c["affine"] else None
    centred = x - x.mean(-1, keepdim=True)
    rstd = 1 / torch.sqrt((centred * centred).mean(-1, keepdim=True) + 1e-5)
    xh = centred * rstd
    y = (xh * w + s["b"].float() if c["affine"] else xh).to(s["x"].dtype)
    if not c["train"]:
        return [y]
    dy = s["dy"].float()
    gw = dy * w if c["affine"] else dy
    dx = rstd * (gw - gw.mean(-1, keepdim=True) - xh * (gw * xh).mean(-1, keepdim=True))
    out = [y, dx.to(y.dtype)]
    if c["affine"]:
        out += [(dy * xh).sum(0).to(s["w"].dtype), dy.sum(0).to(s["b"].dtype)]
    return out


def _plain_linear(s):
    c, dt = s["case"], s["x"].dtype
    x, w = s["x"].float(), s["w"].float()
    z = x @ w.t()
    if c["bias"]:
        z = z + s["b"].float()
    y, slope = (z, None) if c["act"] == "none" else _act(z, c["act"])
    y = (y + s["r"].float() if c["res"] else y).to(dt)
    if not c["train"]:
        return [y]
    dz = s["dy"].float() if slope is None else s["dy"].float() * slope
    out = [y, (dz @ w).to(dt), (dz.t() @ x).to(dt)]
    if c["bias"]:
        out.append(dz.sum(0).to(dt))
    if c["res"]:
        out.append(s["dy"])
    return out


def _turn(x, s, sign):
    pos, at, parts = s["pos"], 0, []
    for axis, (cos, sin) in enumerate(s["tables"]):
        k = cos.shape[1]
        cs, sn = cos[pos[..., axis]], sign * sin[pos[..., axis]]
        if s["case"]["H"]:
            cs, sn = cs.unsqueeze(-2), sn.unsqueeze(-2)
        a, b = x[..., at:at + k], x[..., at + k:at + 2 * k]
        parts += [a * cs - b * sn, a * sn + b * cs]
        at += 2 * k
    return torch.cat(parts + [x[..., at:]], -1)


def _plain_rope(s):
    dt = s["x"].dtype
    out = [_turn(s["x"].float(), s, 1.0).to(dt)]
    if s["case"]["train"]:
        out.append(_turn(s["dy"].float(), s, -1.0).to(dt))
    return out


# ---------------------------------------------------------------------------- one pass
def run(s):
    c = s["case"]
    if not own:
        with torch.no_grad():
            return {"norm": _plain_norm, "linear": _plain_linear, "rope": _plain_rope}[c["op"]](s)
    from pom_b200.operators import apply_rope_axes, layer_norm, linear

    if c["op"] == "norm":
        y = layer_norm(s["x"], s.get("w"), s.get("b"), 1e-5)
    elif c["op"] == "linear":
        y = linear(s["x"], s["w"], s["b"], activation=None if c["act"] == "none" else c["act"], residual=s["r"])
    else:
        y = apply_rope_axes(s["x"], s["pos"], s["tables"], validate=c["checked"])
    if not c["train"]:
        return [y]
    return [y.detach(), *torch.autograd.grad(y, _leaves(s), s["dy"])]


# ---------------------------------------------------------------------------- work and definition
def work(case):
    e, train = (2 if case["dtype"] == "bf16" else 4), case["train"]
    passes = 2 if train else 1  # the input and the output, and their gradients
    if case["op"] == "norm":
        we = 2 if case["wdtype"] == "bf16" else 4
        M, D = case["M"], case["D"]
        return {"bytes": passes * (2 * M * D * e + (2 * D * we if case["affine"] else 0)), "flops": passes * 8 * M * D}
    if case["op"] == "linear":
        M, N, K = case["M"], case["N"], case["K"]
        one = M * K + N * K + M * N + (N if case["bias"] else 0)
        return {"bytes": e * (passes * one + (M * N if case["res"] else 0)), "flops": (3 if train else 1) * 2 * M * N * K}
    n = case["T"] * case["Y"] * case["X"]
    values = case["B"] * n * max(1, case["H"]) * case["D"]
    rows = min(n * (case["B"] if case["own_pos"] else 1), _LEN)
    tables = 8 * rows * (case["st"] + case["sy"] + case["sx"]) + 24 * n * (case["B"] if case["own_pos"] else 1)
    return {"bytes": passes * (2 * values * e) + tables, "flops": passes * 3 * values}


def exact(case, seed):
    s = prepare(case, seed)
    x = s["x"].detach().double()
    dy = s["dy"].double() if case["train"] else None
    if case["op"] == "norm":
        D = case["D"]
        w = s["w"].detach().double() if case["affine"] else torch.ones(D, dtype=torch.float64, device="cuda")
        m = x.sum(1, keepdim=True) / D
        r = (((x - m) ** 2).sum(1, keepdim=True) / D + 1e-5) ** -0.5
        out = [(x - m) * r * w + (s["b"].detach().double() if case["affine"] else 0)]
        if case["train"]:
            n = (x - m) * r
            h = dy * w
            out.append(r / D * (D * h - h.sum(1, keepdim=True) - n * (h * n).sum(1, keepdim=True)))
            if case["affine"]:
                out += [torch.einsum("md,md->d", dy, n), dy.sum(0)]
        return out
    if case["op"] == "linear":
        w = s["w"].detach().double()
        z = torch.einsum("mk,nk->mn", x, w)
        if case["bias"]:
            z += s["b"].detach().double()
        z.requires_grad_(case["train"])
        kind = case["act"]
        with torch.enable_grad():
            if kind == "gelu":
                a = z * torch.special.ndtr(z)
            elif kind == "gelu_tanh":
                a = z * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3))
            elif kind == "silu":
                a = z * torch.sigmoid(z)
            elif kind == "relu":
                a = torch.where(z > 0, z, torch.zeros_like(z))
            else:
                a = z * 1.0
        out = [a.detach() + (s["r"].detach().double() if case["res"] else 0)]
        if case["train"]:
            dz, = torch.autograd.grad(a, z, dy)
            out += [torch.einsum("mn,nk->mk", dz, w), torch.einsum("mn,mk->nk", dz, x)]
            if case["bias"]:
                out.append(torch.einsum("mn->n", dz))
            if case["res"]:
                out.append(dy)
        return out
    # pairs as complex numbers: a rotation is a product with cos + i sin
    turn, at = [], 0
    for axis, (cos, sin) in enumerate(s["tables"]):
        t = torch.complex(cos.double(), sin.double())[s["pos"][..., axis]]
        turn.append((at, cos.shape[1], t.unsqueeze(-2) if case["H"] else t))
        at += 2 * cos.shape[1]

    def rotated(v, conj):
        v = v.clone()
        for lo, k, t in turn:
            z = torch.complex(v[..., lo:lo + k], v[..., lo + k:lo + 2 * k]) * (t.conj() if conj else t)
            v[..., lo:lo + k], v[..., lo + k:lo + 2 * k] = z.real, z.imag
        return v

    return [rotated(x, False)] + ([rotated(dy, True)] if case["train"] else [])
