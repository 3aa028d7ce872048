"""Layer norm, linear and several-axis rotary operators against their definitions in 64 bits.

Every comparison has a bound per element, from the arithmetic: e = 2^-24 is half a step of float32, h half a step of the
output type (2^-8 relative for bf16, e for float32).  A sum of n terms formed in float32 is off by at most n e times the
sum of the terms' magnitudes (2 n e on the tensor cores, whose additions may truncate); every stored value adds h of
itself.  `plus` names what an operand that was stored on the way adds."""
import pytest
import torch

from pom_b200.operators import apply_rope_axes, layer_norm, linear, precompute_freqs_axes

pytestmark = pytest.mark.gpu

E = 2.0 ** -24
BF, F32 = torch.bfloat16, torch.float32
H = {BF: 2.0 ** -8, F32: E}


def rand(*shape, dtype=F32, seed=0, scale=1.0, shift=0.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * scale + shift).to(dtype)


def within(got, want, slack, label):
    """|got - want| <= h |want| + slack, element by element."""
    assert got.shape == want.shape, f"{label}: shape {tuple(got.shape)}, expected {tuple(want.shape)}"
    bad = (got.double() - want).abs() > H[got.dtype] * want.abs() + slack
    bad |= ~torch.isfinite(got) & torch.isfinite(want)
    if bool(bad.any()):
        i = int(bad.flatten().nonzero()[0])
        raise AssertionError(f"{label}: {int(bad.sum())} of {bad.numel()} off, first at {i}: "
                             f"{got.flatten()[i].item()} for {want.flatten()[i].item()}")


# ---------------------------------------------------------------------------- layer norm
def norm_reference(x, w, b, eps, dy):
    x, dy = x.detach().double(), dy.double()
    D = x.shape[-1]
    wd = torch.ones(D, dtype=torch.float64, device=x.device) if w is None else w.detach().double()
    m = x.mean(-1, keepdim=True)
    r = 1 / torch.sqrt(((x - m) ** 2).mean(-1, keepdim=True) + eps)
    xh = (x - m) * r
    y = xh * wd + (0 if b is None else b.detach().double())
    g = dy * wd
    dx = r * (g - g.mean(-1, keepdim=True) - xh * (g * xh).mean(-1, keepdim=True))
    # a thread adds up to 40 values of a row (2 per 1000 in the wide kernels), 9 further additions join the threads
    n = 64 + D / 512
    xe = r * (x.abs() + x.abs().mean(-1, keepdim=True))  # what the error of the mean and of r is relative to
    ye = n * E * (wd.abs() * xe + y.abs())
    dxe = 2 * n * E * r * (g.abs() + g.abs().mean(-1, keepdim=True) + xe * (g * xh).abs().mean(-1, keepdim=True)
                           + xh.abs() * (g.abs() * xe).mean(-1, keepdim=True))
    rows = x.reshape(-1, D).shape[0]
    dw, db = (dy * xh).reshape(-1, D).sum(0), dy.reshape(-1, D).sum(0)
    dwe = (rows + 2 * n) * E * (dy.abs() * xe).reshape(-1, D).sum(0)
    dbe = (rows + 64) * E * dy.abs().reshape(-1, D).sum(0)
    return (y, dx, dw, db), (ye, dxe, dwe, dbe)


def norm_check(x, w, b, dy, eps=1e-5, label=""):
    leaves = [t.detach().clone().requires_grad_(True) if t is not None else None for t in (x, w, b)]
    x0 = leaves[0] if x.is_contiguous() else x.detach().requires_grad_(True)
    y = layer_norm(x0, leaves[1], leaves[2], eps)
    assert y.dtype == x.dtype and y.shape == x.shape
    ins = [t for t in (x0, *leaves[1:]) if t is not None]
    grads = torch.autograd.grad(y, ins, dy)
    want, slack = norm_reference(x, w, b, eps, dy)
    within(y, want[0], slack[0], label + "y")
    with torch.no_grad():
        assert torch.equal(layer_norm(x, w, b, eps), y)
    for got, k, name in zip(grads, (1, 2, 3), ("dx", "dw", "db")):
        assert got.dtype == ins[k - 1].dtype
        within(got, want[k], slack[k], label + name)


# widths: one value, less than a warp, the borders of a warp's, of 128 and of 512 threads' registers, odd ones of each
# kernel, and rows no block can hold
NORM_WIDTHS = [1, 2, 7, 8, 31, 40, 160, 161, 256, 511, 513, 640, 1024, 1152, 1280, 1288, 2048, 2049, 4096, 4104, 8192,
               16392]


@pytest.mark.parametrize("D", NORM_WIDTHS)
@pytest.mark.parametrize("dtype, wdtype", [(BF, BF), (BF, F32), (F32, F32), (F32, BF)])
def test_layer_norm(D, dtype, wdtype):
    M = 37 if D < 4096 else 5
    x = rand(M, D, seed=1, scale=2.0, shift=0.7).to(dtype)
    w, b, dy = rand(D, dtype=wdtype, seed=2, shift=1.0), rand(D, dtype=wdtype, seed=3), rand(M, D, dtype=dtype, seed=4)
    norm_check(x, w, b, dy)
    norm_check(x, None, None, dy, eps=1e-3, label="plain ")
    norm_check(x, w, None, dy, label="no bias ")


@pytest.mark.parametrize("M", [1, 2, 11, 12, 13, 1777, 5000])
@pytest.mark.parametrize("D", [96, 1152, 1536])
def test_layer_norm_rows(M, D):
    x, dy = rand(M, D, dtype=BF, seed=5), rand(M, D, dtype=BF, seed=6)
    norm_check(x, rand(D, dtype=BF, seed=2, shift=1.0), rand(D, dtype=BF, seed=3), dy)


def test_layer_norm_strides():
    base = rand(6, 50, 200, dtype=BF, seed=7)
    w, b = rand(136, dtype=BF, seed=2), rand(136, dtype=BF, seed=3)
    for x in (base[:, :, 8:144], base[:, :, 3:139], base[:, 7:40, 8:144], base.transpose(0, 1)[:, :, 64:], base[0, 0, :136]):
        dy = rand(*x.shape, dtype=BF, seed=8)
        norm_check(x, w, b, dy)
        norm_check(x, w, b, rand(1, dtype=BF, seed=8).expand(x.shape), label="expanded ")


def test_layer_norm_offset_rows_and_constant_rows():
    # a mean of 1000 standard deviations: the variance is taken around the mean, so nothing cancels but x's own steps
    x = rand(9, 1152, seed=9, shift=1000.0)
    norm_check(x, rand(1152, seed=2), rand(1152, seed=3), rand(9, 1152, seed=4))
    x = torch.full((3, 512), 2.5, device="cuda", dtype=BF)
    y = layer_norm(x, None, None, 1e-5)
    assert torch.equal(y, torch.zeros_like(y))


def test_layer_norm_keeps_bad_rows_to_themselves():
    x = rand(8, 1152, dtype=BF, seed=10)
    clean = layer_norm(x)
    x[2, 5], x[5, 1000] = float("inf"), float("nan")
    y = layer_norm(x)
    assert bool(y[2].isnan().all()) and bool(y[5].isnan().all())
    keep = [0, 1, 3, 4, 6, 7]
    assert torch.equal(y[keep], clean[keep])


def test_layer_norm_without_rows():
    x = torch.empty(0, 64, device="cuda", dtype=BF, requires_grad=True)
    w = torch.ones(64, device="cuda", dtype=BF, requires_grad=True)
    y = layer_norm(x, w)
    assert y.shape == (0, 64)
    dx, dw = torch.autograd.grad(y, [x, w], torch.empty_like(y))
    assert dx.shape == (0, 64) and torch.equal(dw, torch.zeros_like(w))


# ---------------------------------------------------------------------------- linear
ACTS = [None, "gelu", "gelu_tanh", "silu", "relu"]


def act_reference(z, kind):
    z = z.detach().requires_grad_(True)
    if kind is None:
        y = z * 1.0
    elif kind == "gelu":
        y = z * torch.special.ndtr(z)
    elif kind == "gelu_tanh":
        y = torch.nn.functional.gelu(z, approximate="tanh")
    elif kind == "silu":
        y = z * torch.sigmoid(z)
    else:
        y = torch.relu(z)
    s, = torch.autograd.grad(y.sum(), z)
    return y.detach(), s


def linear_check(x, w, b, r, act, dy, label=""):
    dt = x.dtype
    h = H[dt]
    ins = [t.detach().requires_grad_(True) for t in (x, w, b, r) if t is not None]
    it = iter(ins)
    args = [next(it) if t is not None else None for t in (x, w, b, r)]
    y = linear(args[0], args[1], args[2], activation=act, residual=args[3])
    assert y.dtype == dt and y.shape == (*x.shape[:-1], w.shape[0])
    grads = torch.autograd.grad(y, ins, dy)
    with torch.no_grad():
        assert torch.equal(linear(x, w, b, activation=act, residual=r), y), label + "untracked"
    N, K = w.shape
    xd, wd, g = (t.detach().double().reshape(-1, t.shape[-1]) for t in (x, w, dy))
    M = xd.shape[0]
    z = xd @ wd.t() + (0 if b is None else b.detach().double())
    ze = 2 * (K + 8) * E * (xd.abs() @ wd.abs().t() + (0 if b is None else b.detach().double().abs()))
    a, s = act_reference(z, act)
    # every activation grows by at most 1.13 per unit; its own evaluation is good to 16 half steps of |z| + 1
    ye = 1.13 * ze + (0 if act is None else 16 * E * (z.abs() + 1)) + E * a.abs()
    want = a
    if r is not None:
        want = a + r.detach().double().reshape(M, N)
    within(y.detach().reshape(M, N), want, ye + E * want.abs(), label + "y")
    # the slope, which changes by at most 0.8 per unit of z (relu: any amount within ze of 0), is taken at the stored z
    se = 0 if act is None else 0.8 * (ze + h * z.abs()) + 16 * E * (z.abs() + 1)
    if act == "relu":
        se = se + (z.abs() <= ze).double()
    dz = g * s
    dze = g.abs() * se if act is not None else torch.zeros_like(g)
    stored = dze + (h * dz.abs() if act is not None else 0)  # dz is rounded before the products
    out = dict(x=(dz @ wd, stored @ wd.abs() + 2 * (N + 8) * E * (dz.abs() @ wd.abs())),
               w=(dz.t() @ xd, stored.t() @ xd.abs() + 2 * (M + 8) * E * (dz.abs().t() @ xd.abs())))
    names = ["x", "w"]
    if b is not None:
        out["b"] = (dz.sum(0), dze.sum(0) + (M + 64) * E * dz.abs().sum(0))
        names.append("b")
    if r is not None:
        out["r"] = (g, torch.zeros_like(g))
        names.append("r")
    for got, name, ref in zip(grads, names, ins):
        assert got.dtype == ref.dtype and got.shape == ref.shape
        ww, slack = out[name]
        within(got.reshape(ww.shape), ww, slack + E * ww.abs(), f"{label}d{name}")


def linear_inputs(M, K, N, dtype, bias_dtype=None, seed=0):
    x, w = rand(M, K, dtype=dtype, seed=seed), rand(N, K, dtype=dtype, seed=seed + 1, scale=K ** -0.5)
    b, r = rand(N, dtype=bias_dtype or dtype, seed=seed + 2, scale=0.3), rand(M, N, dtype=dtype, seed=seed + 3)
    return x, w, b, r, rand(M, N, dtype=dtype, seed=seed + 4)


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("M", [1, 5, 16, 17, 40, 64, 65, 300])
def test_linear_activations(M, dtype, act):
    x, w, b, r, dy = linear_inputs(M, 136, 200, dtype)
    for bias, res in ((None, None), (b, None), (None, r), (b, r)):
        linear_check(x, w, bias, res, act, dy, label=f"bias {bias is not None}, residual {res is not None}: ")


@pytest.mark.parametrize("K, N", [(8, 8), (1, 1), (7, 9), (33, 17), (16, 600), (600, 16), (1152, 264), (264, 1160), (520, 2600)])
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("M", [1, 33, 129, 1000])
def test_linear_sizes(M, K, N, dtype):
    x, w, b, r, dy = linear_inputs(M, K, N, dtype, seed=10)
    linear_check(x, w, b, r, "gelu", dy)
    linear_check(x, w, b, None, None, dy, label="plain ")


@pytest.mark.parametrize("act", [None, "gelu", "relu"])
@pytest.mark.parametrize("M, K, N", [(65, 1096, 136), (130, 2056, 264), (300, 1160, 1096), (1000, 136, 72), (2049, 72, 136),
                                     (200, 1000, 1160), (500, 2312, 520), (1100, 2120, 1032), (2000, 4104, 1000), (129, 264, 120),
                                     (1000, 3080, 1160), (385, 4616, 264), (513, 1032, 2056)])
def test_linear_products_cut_along_their_sum(M, K, N, act):
    """Few output tiles and a long sum: the product and the data gradient run on clusters of two to eight blocks, the
    weight gradient in slabs."""
    x, w, b, r, dy = linear_inputs(M, K, N, BF, F32 if act == "gelu" else BF, seed=60)
    linear_check(x, w, b, r, act, dy)
    linear_check(x, w, None, None, act, dy, label="plain ")


def test_linear_bias_types_and_strides():
    x, w, b, r, dy = linear_inputs(200, 256, 320, BF, F32, seed=20)
    linear_check(x, w, b, r, "silu", dy)
    linear_check(x[:9], w, b, r[:9], "silu", dy[:9])
    wide = rand(200, 400, dtype=BF, seed=25)
    tall = rand(320, 300, dtype=BF, seed=26)
    for lo in (8, 16, 3):  # aligned rows of a wider matrix, and rows that have to be copied
        for m in (200, 12):
            linear_check(wide[:m, lo:lo + 256], tall[:, lo:lo + 256], b, r[:m], "gelu", dy[:m], label=f"{lo} ")
    linear_check(wide.t()[:256].t(), w, b, r.t().contiguous().t(), None, dy.t().contiguous().t())
    linear_check(x.view(4, 50, 256), w, b, r.view(4, 50, 320), "gelu", dy[:1, :1].expand(200, 320).reshape(4, 50, 320))
    linear_check(x.view(4, 50, 256), w, b, None, "gelu", dy[:1, :1].unsqueeze(0).expand(4, 50, 320))


def test_linear_only_some_gradients():
    x, w, b, r, dy = linear_inputs(150, 64, 72, BF, seed=30)
    want = None
    for which in ("xwbr", "x", "w", "b", "r", "xw", "wb"):
        ins = {k: t.detach().clone().requires_grad_(k in which) for k, t in zip("xwbr", (x, w, b, r))}
        y = linear(ins["x"], ins["w"], ins["b"], activation="gelu", residual=ins["r"])
        got = dict(zip(which, torch.autograd.grad(y, [ins[k] for k in which], dy)))
        want = want or got
        for k in which:
            assert torch.equal(got[k], want[k]), (which, k)


def test_linear_few_rows_of_any_width():
    """Untracked products of up to 32 rows take any N without a padded copy; a residual view of any alignment."""
    for M, K in ((1, 72), (16, 72), (17, 72), (32, 72), (33, 72), (32, 2048), (16, 2056), (17, 2056), (32, 2049)):
        for N in (1, 7, 130, 2369):
            x, w, b, r, _ = linear_inputs(M, K, N, BF, F32, seed=45)
            wide = rand(M, N + 3, dtype=BF, seed=46)
            for res in (None, r, wide[:, 3:]):
                with torch.no_grad():
                    y = linear(x, w, b, activation="gelu", residual=res)
                z = x.double() @ w.double().t() + b.double()
                ze = 2 * (K + 8) * E * (x.double().abs() @ w.double().abs().t() + b.double().abs())
                want = act_reference(z, "gelu")[0] + (0 if res is None else res.double())
                within(y, want, 1.13 * ze + 16 * E * (z.abs() + 1) + E * want.abs(), f"{M} {N}")


@pytest.mark.parametrize("M", [16, 17, 24, 32, 33])
@pytest.mark.parametrize("K, N", [(2048, 200), (2056, 200), (2056, 205), (4608, 72)])
def test_linear_few_rows_long_sums(K, N, M):
    x, w, b, r, dy = linear_inputs(M, K, N, BF, F32, seed=47)
    linear_check(x, w, b, r, "silu", dy)


def test_linear_without_rows():
    for dtype in (BF, F32):
        x = torch.empty(2, 0, 64, device="cuda", dtype=dtype, requires_grad=True)
        w, b = rand(24, 64, dtype=dtype).requires_grad_(True), rand(24, dtype=dtype).requires_grad_(True)
        y = linear(x, w, b, activation="relu")
        assert y.shape == (2, 0, 24)
        dx, dw, db = torch.autograd.grad(y, [x, w, b], torch.empty_like(y))
        assert dx.shape == x.shape and not dw.any() and not db.any()


def test_linear_far_values():
    """Saturated activations: far below 0 they and their slopes vanish, far above they pass; no NaN from an overflow."""
    z = torch.tensor([-3e4, -200.0, -40.0, -9.0, 0.0, 9.0, 40.0, 200.0, 3e4], device="cuda")
    for dtype in (BF, F32):
        zz = z.to(dtype)
        for m in (9, 90):
            x = zz.repeat(m // 9)[:, None].expand(m, 8).contiguous()
            x[:, 1:] = 0
            w = torch.eye(8, device="cuda", dtype=dtype)
            for act in ACTS[1:]:
                x.requires_grad_(True)
                y = linear(x, w, activation=act)
                dx, = torch.autograd.grad(y, x, torch.ones_like(y))
                x.requires_grad_(False)
                big = zz.repeat(m // 9).abs() >= 40
                pos = zz.repeat(m // 9) > 0
                assert torch.equal(y[big & pos, 0], x[big & pos, 0]) and (y[big & ~pos, 0].abs() < 1e-6).all()
                assert (dx[big & pos, 0] == 1).all() and (dx[big & ~pos, 0].abs() < 1e-6).all()


def test_linear_keeps_bad_values_to_their_rows_and_columns():
    for m in (10, 200):
        x, w, b, _, _ = linear_inputs(m, 128, 264, BF, seed=40)
        clean = linear(x, w, b, activation="relu")
        x[3, 7] = float("nan")
        w[11, 5] = float("inf")
        y = linear(x, w, b, activation="relu")
        assert bool(y[3].isnan().all())
        rows = [i for i in range(m) if i != 3]
        cols = [i for i in range(264) if i != 11]
        assert torch.equal(y[rows][:, cols], clean[rows][:, cols])


def test_linear_autocast():
    x, w, b, r, dy = linear_inputs(80, 64, 96, F32, seed=50)
    ins = [t.requires_grad_(True) for t in (x, w, b, r)]
    with torch.autocast("cuda", BF):
        y = linear(x, w, b, activation="gelu", residual=r)
    assert y.dtype == BF
    grads = torch.autograd.grad(y, ins, dy.to(BF))
    assert all(g.dtype == F32 for g in grads)
    with torch.no_grad():
        assert torch.equal(y, linear(x.to(BF), w.to(BF), b, activation="gelu", residual=r.to(BF)))


# ---------------------------------------------------------------------------- rotary positions of several axes
def rope_reference(x, pos, tables, conj):
    x = x.detach().double()
    y, mag, at = x.clone(), x.abs(), 0
    for a, (c, s) in enumerate(tables):
        k = c.shape[1]
        z = torch.complex(c.double(), s.double())[pos[..., a]]
        z = z.unsqueeze(-2) if x.dim() == 4 else z
        v = torch.complex(x[..., at:at + k], x[..., at + k:at + 2 * k]) * (z.conj() if conj else z)
        y[..., at:at + k], y[..., at + k:at + 2 * k] = v.real, v.imag
        both = x[..., at:at + k].abs() + x[..., at + k:at + 2 * k].abs()
        mag[..., at:at + k] = mag[..., at + k:at + 2 * k] = both
        at += 2 * k
    return y, 3 * E * mag


def rope_check(x, pos, tables, label=""):
    ref_tables = [(c.cuda(), s.cuda()) for c, s in tables]
    x = x.detach().requires_grad_(True)
    y = apply_rope_axes(x, pos, tables)
    assert y.dtype == x.dtype and y.shape == x.shape
    within(y.detach(), *rope_reference(x, pos, ref_tables, False), label + "y")
    dy = rand(*x.shape, dtype=x.dtype, seed=99)
    for g in (dy, dy.transpose(0, 1).contiguous().transpose(0, 1), dy[:1, :1].expand(x.shape)):
        dx, = torch.autograd.grad(y, x, g, retain_graph=True)
        within(dx, *rope_reference(g, pos, ref_tables, True), label + "dx")
    with torch.no_grad():
        assert torch.equal(apply_rope_axes(x, pos, tables, validate=False), y)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("pairs, extra", [((8,), 0), ((8, 16, 24), 0), ((2, 4, 6), 0), ((1, 3, 5), 0), ((1,), 0), ((8, 8, 8), 16),
                                          ((8, 8, 8), 5), ((3, 2), 1), ((16, 8, 8, 24), 8), ((384, 384, 384), 0)])
@pytest.mark.parametrize("heads", [0, 1, 3])
def test_rope_axes(pairs, extra, heads, dtype):
    B, N, D = 3, 41, 2 * sum(pairs) + extra
    tables = precompute_freqs_axes(pairs, [20 + 7 * i for i in range(len(pairs))])
    g = torch.Generator(device="cuda").manual_seed(5)
    x = rand(B, N, *((heads,) if heads else ()), D, dtype=dtype, seed=1)
    for shape in ((N,), (B, N)):
        pos = torch.stack([torch.randint(0, len(c), shape, generator=g, device="cuda") for c, _ in tables], -1)
        rope_check(x, pos, tables, label=f"{shape} ")


def test_rope_axes_strides_and_sizes():
    tables = [(c.cuda(), s.cuda()) for c, s in precompute_freqs_axes((16, 8), (64, 64))]
    base = rand(4, 60, 3, 80, dtype=BF, seed=2)
    pos = torch.randint(0, 64, (60, 2), device="cuda")
    for x in (base, base[..., 8:72], base[..., 3:55], base[:, ::2], base.transpose(1, 2).contiguous().transpose(1, 2),
              base[:, :1], base[:1], base[:, :, 1], base[0:0], base.expand(4, 60, 3, 80), base[:1].expand(5, 60, 3, 80)):
        rope_check(x, pos[:x.shape[1]] if x.shape[1] != 30 else pos[::2], tables)
    x = rand(2, 3001, 96, dtype=BF, seed=3)  # more work than the grid has threads
    rope_check(x, torch.randint(0, 64, (3001, 2), device="cuda"), tables)
    rope_check(x, torch.randint(0, 64, (2, 3001, 2), device="cuda").to(torch.int32).long(), tables)


def test_rope_axes_equals_the_two_axis_form():
    from pom_b200.operators import apply_rope_2d

    tables = [(c.cuda(), s.cuda()) for c, s in precompute_freqs_axes((32, 32), (16, 16))]
    x = rand(2, 256, 128, seed=4)
    hw = torch.stack([torch.arange(256) // 16, torch.arange(256) % 16], -1).cuda()
    a = apply_rope_axes(x, hw, tables)
    b = apply_rope_2d(x, hw, *tables[0], *tables[1])
    assert (a - b).abs().max() <= 8 * E * x.abs().max()


def test_rope_axes_positions_outside_the_tables():
    tables = [(c.cuda(), s.cuda()) for c, s in precompute_freqs_axes((8, 8), (10, 12))]
    x = rand(2, 5, 40, dtype=BF, seed=6)
    pos = torch.randint(0, 10, (5, 2), device="cuda")
    good = apply_rope_axes(x, pos, tables)
    for bad in (-1, 12, 1 << 40, -(1 << 62)):
        p = pos.clone()
        p[3, 1] = bad
        with pytest.raises(IndexError, match="axis 1"):
            apply_rope_axes(x, p, tables)
        y = apply_rope_axes(x, p, tables, validate=False)
        assert bool(y[:, 3, 16:32].isnan().all())
        y[:, 3, 16:32] = good[:, 3, 16:32]
        assert torch.equal(y, good)
    p = pos.clone()
    apply_rope_axes(x, p, tables)
    p[0, 0] = 10  # an update in place is seen
    with pytest.raises(IndexError, match="axis 0"):
        apply_rope_axes(x, p, tables)
    # more rows than one block looks through
    many = torch.zeros(70000, 2, dtype=torch.int64, device="cuda")
    x = rand(1, 70000, 32, dtype=BF, seed=6)
    assert torch.equal(apply_rope_axes(x, many, tables), x)
    for at, axis, bad in ((69999, 0, 10), (0, 1, 12), (40000, 1, -1), (123, 0, -(1 << 62)), (5, 1, 1 << 62)):
        p = many.clone()
        p[at, axis] = bad
        with pytest.raises(IndexError, match=f"axis {axis}"):
            apply_rope_axes(x, p, tables)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        with pytest.raises(RuntimeError, match="validate=False"):
            apply_rope_axes(x, many, tables)
        y = apply_rope_axes(x, many, tables, validate=False)
    g.replay()
    assert torch.equal(y, x)


def test_rope_axes_notices_positions_that_change_before_backward():
    tables = [(c.cuda(), s.cuda()) for c, s in precompute_freqs_axes((8, 8), (10, 12))]
    x = rand(2, 5, 40, seed=6).requires_grad_(True)
    pos = torch.randint(0, 9, (5, 2), device="cuda")
    y = apply_rope_axes(x, pos, tables)
    pos.add_(1)
    with pytest.raises(RuntimeError, match="inplace"):
        torch.autograd.grad(y.sum(), x)
    with pytest.raises(ValueError, match="gradient"):
        apply_rope_axes(x, pos, [(tables[0][0].clone().requires_grad_(True), tables[0][1]), tables[1]])


# ---------------------------------------------------------------------------- all three: streams, graphs, repetition
def block_pass(t):
    """The chain that a block runs, and all gradients."""
    h = layer_norm(t["x"], t["nw"], t["nb"])
    h = apply_rope_axes(h, t["pos"], t["tables"], validate=False)
    u = linear(h, t["w1"], t["b1"], activation="gelu")
    y = linear(u, t["w2"], t["b2"], residual=t["x"])
    grads = torch.autograd.grad(y, [t[k] for k in ("x", "nw", "nb", "w1", "b1", "w2", "b2")], t["dy"])
    return [y.detach(), *grads]


def block_tensors(dtype, B=2, N=96, D=192, seed=70):
    t = dict(x=rand(B, N, D, dtype=dtype, seed=seed), nw=rand(D, dtype=dtype, seed=seed + 1, shift=1.0, scale=0.2),
             nb=rand(D, dtype=dtype, seed=seed + 2, scale=0.2), w1=rand(4 * D, D, dtype=dtype, seed=seed + 3, scale=D ** -0.5),
             b1=rand(4 * D, dtype=dtype, seed=seed + 4, scale=0.2),
             w2=rand(D, 4 * D, dtype=dtype, seed=seed + 5, scale=(4 * D) ** -0.5), b2=rand(D, dtype=dtype, seed=seed + 6, scale=0.2))
    t = {k: v.requires_grad_(True) for k, v in t.items()}
    t["dy"] = rand(B, N, D, dtype=dtype, seed=seed + 7)
    i = torch.arange(N, device="cuda")
    t["pos"] = torch.stack([i // 32, i // 8 % 4, i % 8], -1)
    t["tables"] = [(c.cuda(), s.cuda()) for c, s in precompute_freqs_axes((D // 8, D // 8, D // 4), (8, 8, 8))]
    return t


@pytest.mark.parametrize("dtype", [BF, F32])
def test_a_block_against_64_bits(dtype):
    t = block_tensors(dtype)
    got = block_pass(t)
    d = {k: v.detach().double().requires_grad_(True) for k, v in t.items() if k in ("x", "nw", "nb", "w1", "b1", "w2", "b2")}
    h = torch.nn.functional.layer_norm(d["x"], (192,), d["nw"], d["nb"])
    parts, at = [], 0
    for a, (c, s) in enumerate(t["tables"]):
        k = c.shape[1]
        cs, sn = c.double()[t["pos"][:, a]], s.double()[t["pos"][:, a]]
        p, q = h[..., at:at + k], h[..., at + k:at + 2 * k]
        parts += [p * cs - q * sn, p * sn + q * cs]
        at += 2 * k
    h = torch.cat([*parts, h[..., at:]], -1)
    u = torch.nn.functional.gelu(h @ d["w1"].t() + d["b1"])
    y = u @ d["w2"].t() + d["b2"] + d["x"]
    want = [y, *torch.autograd.grad(y, list(d.values()), t["dy"].double())]
    # up to seven stored values on the way, each off by at most half a step, mostly independently: 7^(1/2) < 3 of them in
    # the 2-norm; float32: sums of up to 768 terms, 768^(1/2) < 28 half steps per product, four products
    tol = 3 * H[BF] if dtype == BF else 4 * 28 * E
    for i, (a, b) in enumerate(zip(got, want)):
        rel = ((a.double() - b).norm() / b.norm()).item()
        assert rel <= tol, (i, rel)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_same_bits_every_time_on_any_stream_and_from_graphs(dtype):
    t = block_tensors(dtype, B=3, N=352)
    t["pos"] = t["pos"] % 8
    want = block_pass(t)
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(block_pass(t), want))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = block_pass(t)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    # two captured passes, replayed at the same time: they share no workspace
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(block_pass(t))
        graphs.append(g)
    torch.cuda.synchronize()
    for _ in range(3):
        with torch.cuda.stream(side):
            graphs[0].replay()
        graphs[1].replay()
        torch.cuda.synchronize()
        for out in outs:
            assert all(torch.equal(a, b) for a, b in zip(out, want))
            for o in out:
                o.zero_()
        torch.cuda.synchronize()


def test_more_float32_rows_than_one_launch_takes():
    M = 65535 * 64 + 70
    x, w = rand(M, 8, seed=1), rand(8, 8, seed=2)
    x.requires_grad_(True)
    y = linear(x, w, activation="relu")
    dx, = torch.autograd.grad(y, x, torch.ones_like(y))
    with torch.no_grad():
        for sl in (slice(0, 5), slice(M - 100, M), slice(65535 * 64 - 3, 65535 * 64 + 3)):
            z = x[sl].double() @ w.double().t()
            ze = 2 * 16 * E * (x[sl].double().abs() @ w.double().abs().t())
            within(y[sl], z.clamp(min=0), ze, "y")
            near = ((z.abs() <= ze).double()) @ w.double().abs()
            within(dx[sl], (z > 0).double() @ w.double(), near + 32 * E * w.double().abs().sum(0), "dx")


def test_vectors_and_keyword_arguments():
    x, w, b, r, _ = linear_inputs(1, 64, 40, BF, seed=97)
    y = linear(x=x[0], weight=w, bias=b, activation="silu", residual=r[0])
    assert torch.equal(y, linear(x, w, b, activation="silu", residual=r)[0])
    assert torch.equal(layer_norm(x=x[0], weight=x[0].abs()), layer_norm(x, x[0].abs())[0])


def test_gradients_against_differences():
    """The float32 gradients along random directions against central differences of the float64 definition."""
    x, w, b, r, dy = linear_inputs(70, 48, 40, F32, seed=80)
    ins = [t.requires_grad_(True) for t in (x, w, b, r)]
    for act in ("gelu", "gelu_tanh", "silu"):
        y = linear(x, w, b, activation=act, residual=r)
        grads = torch.autograd.grad(y, ins, dy)

        def value(*t):
            return ((act_reference(t[0] @ t[1].t() + t[2], act)[0] + t[3]) * dy.double()).sum()

        base = [t.detach().double() for t in ins]
        for i, g in enumerate(grads):
            v = rand(*g.shape, seed=90 + i).double()
            step = 1e-5
            up, down = list(base), list(base)
            up[i], down[i] = base[i] + step * v, base[i] - step * v
            slope = (value(*up) - value(*down)) / (2 * step)
            # float32 gradients: each element within 200 E of sums of at most 70 terms; differences: step^2
            size = (g.double().abs() * v.abs()).sum()
            assert abs(slope - (g.double() * v).sum()) <= 400 * E * size + 1e-7 * abs(slope) + 1e-6


def test_double_backward_is_refused():
    x, w, b, r, dy = linear_inputs(8, 16, 16, F32, seed=95)
    x.requires_grad_(True)
    for y in (linear(x, w, b, activation="gelu"), layer_norm(x)):
        g, = torch.autograd.grad(y.sum(), x, create_graph=True)
        with pytest.raises(RuntimeError):
            torch.autograd.grad(g.sum(), x)
