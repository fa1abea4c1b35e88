"""The matrix operators on the GPU against plain 64-bit implementations.

Tolerances.

* A linear layer's y is its 64-bit value rounded once: half an ulp of the
  output type (U: 2^-8 bf16, 2^-11 fp16, relative), plus the fp32 sum's error,
  at most (K + 16) 2^-22 of the sum of the terms' magnitudes (tensor cores may
  truncate each addition). Activations are Lipschitz with constant 1.13 and
  their own fp32 error is a few 2^-22 of |z|.
* dz carries one more half ulp, the derivative's fixed-point step (2^-15 |dy|)
  and act'' (at most 1.2) times z's own error; dx and dw are linear in it.
* An orthogonalised matrix meets 15 roundings to 11 bits in five steps (X, A
  and the polynomial; relative 2^-12 each), carried on by factors around one:
  6e-3 of the 2-norm covers them added up with a factor 1.6. (With 8-bit
  operands the same sum is 8 times larger, so the bound tells them apart.)
  Results in bf16 add a half ulp of 2^-8 per element.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
QUINTIC = (3.4445, -4.7750, 2.0315)
ORTHO_TOL = 6e-3
ACTS = [None, "relu", "gelu", "gelu_tanh", "silu"]


@pytest.fixture(autouse=True)
def _status_clean():
    from turboadam_b200 import matrix

    yield
    assert matrix.read_status() == 0


def act64(z, kind):
    if kind == "relu":
        return z.clamp(min=0), (z > 0).double()
    if kind == "gelu":
        c = 0.5 * torch.special.erfc(-z / math.sqrt(2))
        return z * c, c + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    if kind == "gelu_tanh":
        k = math.sqrt(2 / math.pi)
        t = torch.tanh(k * (z + 0.044715 * z ** 3))
        d = 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * k * (1 + 3 * 0.044715 * z * z)
        return 0.5 * z * (1 + t), d
    if kind == "silu":
        s = torch.sigmoid(z)
        return z * s, s * (1 + z * (1 - s))
    return z, torch.ones_like(z)


def make_linear(tokens, fan_in, fan_out, dtype, layout="oi", bias=True, residual=True, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def rand(*s):
        return torch.randn(*s, device="cuda", generator=g)

    w = rand(fan_out, fan_in) / math.sqrt(max(fan_in, 1))
    w = w.to(dtype) if layout == "oi" else w.t().contiguous().to(dtype).t()
    return dict(x=rand(tokens, fan_in).to(dtype), w=w,
                b=rand(fan_out).mul(0.1).to(dtype) if bias else None,
                r=rand(tokens, fan_out).to(dtype) if residual else None,
                dy=rand(tokens, fan_out).to(dtype))


def within(got, want, tol, what):
    err = (got.double() - want).abs()
    over = err - tol
    assert bool((over <= 0).all()), (f"{what}: off by {err[over > 0].max().item():.3e}, "
                                     f"{over.max().item():.3e} over its bound, at "
                                     f"{int((over > 0).sum())} of {err.numel()}")


def check_linear(c, act, grads=True):
    from turboadam_b200 import linear_act

    dtype = c["x"].dtype
    u = U[dtype]
    leaves = {k: c[k].detach().requires_grad_(grads) for k in "xwbr" if c[k] is not None}
    y = linear_act(leaves["x"], leaves["w"], leaves.get("b"), activation=act,
                   residual=leaves.get("r"))
    assert y.dtype == dtype and y.shape == c["dy"].shape
    x, w, dy = c["x"].double(), c["w"].double(), c["dy"].double()
    k = x.shape[1]
    z, mag = x @ w.t(), x.abs() @ w.abs().t()
    if c["b"] is not None:
        z, mag = z + c["b"].double(), mag + c["b"].double().abs()
    z_err = (k + 16) * 2.0 ** -22 * mag
    v, d = act64(z, act)
    r = c["r"].double() if c["r"] is not None else torch.zeros_like(z)
    want = v + r
    exact_err = 1.13 * z_err + 2.0 ** -21 * (z.abs() + r.abs())
    within(y.detach(), want, u * want.abs() * (1 + u) + exact_err * (1 + u) + 2.0 ** -25, "y")
    if not grads:
        return
    got = dict(zip(leaves, torch.autograd.grad(y, list(leaves.values()), c["dy"])))
    dz = dy * d
    if act == "relu":  # the step: an argument within its own error of zero may take either side
        d_err = (z.abs() <= z_err).double()
    else:
        d_err = (2.0 ** -15 + 2.0 ** -20 + 1.2 * z_err) if act else torch.zeros_like(z)
    dz_fp32 = dy.abs() * d_err + 2.0 ** -23 * dz.abs()
    dz_err = dz_fp32 + (u * (dz.abs() + dz_fp32) if act else 0) + 2.0 ** -25
    t, o = dy.shape
    mag = dz.abs() @ w.abs()
    tol = dz_err @ w.abs() + (o + 16) * 2.0 ** -22 * mag
    want = dz @ w
    within(got["x"], want, tol * (1 + u) + u * want.abs() + 2.0 ** -25, "dx")
    mag = dz.abs().t() @ x.abs()
    tol = dz_err.t() @ x.abs() + (t + 16) * 2.0 ** -22 * mag
    want = dz.t() @ x
    within(got["w"], want, tol * (1 + u) + u * want.abs() + 2.0 ** -25, "dw")
    assert got["w"].stride() == c["w"].stride() or min(c["w"].shape) == 1
    if "b" in got:
        want = dz.sum(0)
        tol = dz_fp32.sum(0) + (t + 16) * 2.0 ** -23 * dz.abs().sum(0)
        within(got["b"], want, tol * (1 + u) + U[c["b"].dtype] * want.abs() + 2.0 ** -25, "db")
    if "r" in got:
        assert torch.equal(got["r"], c["dy"])


# tile edges (128, 256), k blocks (64), single tokens, odd sizes, sizes of one
LINEAR_SIZES = [(1, 1, 1), (1, 64, 128), (1, 1000, 2304), (2, 65, 7), (3, 8, 257), (8, 768, 768),
                (9, 768, 129), (127, 63, 127), (128, 64, 128), (129, 72, 130), (255, 1, 300),
                (256, 256, 256), (257, 1001, 33), (640, 4096, 96), (1000, 129, 1003),
                (2048, 768, 2304)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("tokens,fan_in,fan_out", LINEAR_SIZES)
def test_linear_sizes(tokens, fan_in, fan_out, dtype):
    act = ACTS[(tokens + fan_in + fan_out) % 5]
    layout = "oi" if (tokens + fan_out) % 2 else "io"
    check_linear(make_linear(tokens, fan_in, fan_out, dtype, layout), act)


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("bias,residual", [(False, False), (True, False), (False, True)])
def test_linear_epilogues(act, bias, residual):
    check_linear(make_linear(200, 96, 272, torch.bfloat16, bias=bias, residual=residual), act)


def test_linear_large_tiles():
    """Sizes that take the 256 x 256 tiles of SM pairs, with ragged edges, in both layouts."""
    for layout in ("oi", "io"):
        check_linear(make_linear(4100, 520, 4104, torch.bfloat16, layout), "silu")
    check_linear(make_linear(4099, 328, 4097, torch.float16, "oi"), "gelu")


@pytest.mark.parametrize("act", ACTS)
def test_linear_no_gradients(act):
    c = make_linear(33, 200, 120, torch.bfloat16)
    check_linear(c, act, grads=False)


def test_linear_float32_bias_and_leading_dims():
    from turboadam_b200 import linear_act

    c = make_linear(6 * 35, 48, 56, torch.bfloat16)
    b = c["b"].float() * 1.001
    y = linear_act(c["x"].view(6, 35, 48), c["w"], b, activation="gelu",
                   residual=c["r"].view(6, 35, 56))
    assert y.shape == (6, 35, 56)
    z = c["x"].double() @ c["w"].double().t() + b.double()
    want = act64(z, "gelu")[0] + c["r"].double()
    within(y.view(210, 56), want, 2.0 ** -8 * want.abs() + 1e-4, "y")
    one = linear_act(c["x"][0], c["w"], b)
    assert one.shape == (56,)


def test_linear_strided_operands():
    """Column slices, row strides that are not 16-byte multiples, transposed tokens, offsets."""
    from turboadam_b200 import linear_act

    g = torch.Generator(device="cuda").manual_seed(1)
    big = torch.randn(300, 211, device="cuda", generator=g).bfloat16()
    wide = torch.randn(150, 400, device="cuda", generator=g).bfloat16()
    for x in (big[:, 3:99], big[1:, :96], big[::2, 8:104], big.t()[:96, :].t(),
              big[:, :96].t().contiguous().t(), big[:1, :96].expand(40, 96)):
        for w in (wide[:, 1:97], wide[::3, :96], wide[:, 100:196], wide[:96, :].t(),
                  wide[:96, 7:90].t()):
            r = torch.randn(x.shape[0], 2 * w.shape[0] + 1, device="cuda", generator=g)
            r = r.bfloat16()[:, 1:1 + w.shape[0]]
            y = linear_act(x, w, residual=r)
            want = x.double() @ w.double().t() + r.double()
            mag = x.double().abs() @ w.double().abs().t()
            within(y, want, 2.0 ** -8 * want.abs() + 112 * 2.0 ** -22 * mag + 1e-6, "y")


def test_linear_gradient_of_strided_output():
    """dy arrives expanded, transposed or with odd strides."""
    from turboadam_b200 import linear_act

    c = make_linear(65, 40, 24, torch.bfloat16, residual=False)
    for dy in (torch.ones(1, 1, device="cuda").bfloat16().expand(65, 24),
               c["dy"].t().contiguous().t(), torch.cat([c["dy"]] * 2, 1)[:, 3:27]):
        x, w = c["x"].detach().requires_grad_(True), c["w"].detach().requires_grad_(True)
        gx, gw = torch.autograd.grad(linear_act(x, w), (x, w), dy)
        wx, ww = dy.double() @ w.double(), dy.double().t() @ x.double()
        within(gx, wx.detach(), 2.0 ** -8 * wx.abs() + 1e-4, "dx")
        within(gw, ww.detach(), 2.0 ** -8 * ww.abs() + 1e-4, "dw")


def test_linear_empty():
    from turboadam_b200 import linear_act

    bf = dict(device="cuda", dtype=torch.bfloat16)
    assert linear_act(torch.empty(0, 8, **bf), torch.empty(5, 8, **bf)).shape == (0, 5)
    assert linear_act(torch.empty(3, 8, **bf), torch.empty(0, 8, **bf)).shape == (3, 0)
    b, r = torch.randn(5, **bf), torch.randn(3, 5, **bf)
    y = linear_act(torch.empty(3, 0, **bf), torch.empty(5, 0, **bf), b, residual=r)
    assert torch.equal(y, (b.float() + r.float()).bfloat16())
    x = torch.empty(0, 8, **bf).requires_grad_(True)
    w = torch.randn(5, 8, **bf).requires_grad_(True)
    b = torch.randn(5, **bf).requires_grad_(True)
    gx, gw, gb = torch.autograd.grad(linear_act(x, w, b, activation="relu"), (x, w, b),
                                     torch.empty(0, 5, **bf))
    assert gx.shape == (0, 8) and gw.abs().sum() == 0 and gb.abs().sum() == 0


def test_linear_some_gradients():
    from turboadam_b200 import linear_act

    c = make_linear(70, 32, 48, torch.bfloat16)
    full = [c[k].detach().requires_grad_(True) for k in "xwbr"]
    want = torch.autograd.grad(linear_act(full[0], full[1], full[2], "gelu", full[3]), full,
                               c["dy"])
    for i in range(4):
        part = [c[k].detach().requires_grad_(j == i) for j, k in enumerate("xwbr")]
        got, = torch.autograd.grad(linear_act(part[0], part[1], part[2], "gelu", part[3]),
                                   [part[i]], c["dy"])
        assert torch.equal(got, want[i])


def test_linear_non_finite():
    """Infinities and NaN go where the formulas send them, and nowhere else."""
    from turboadam_b200 import linear_act

    inf, nan = float("inf"), float("nan")
    for act in ACTS:
        x = torch.zeros(130, 16, device="cuda", dtype=torch.bfloat16)
        x[1, 0], x[2, 0], x[3, 0] = inf, -inf, nan
        x.requires_grad_(True)
        w = torch.zeros(20, 16, device="cuda", dtype=torch.bfloat16)
        w[:, 0] = 1
        b = torch.full((20,), 0.5, device="cuda", dtype=torch.bfloat16)
        y = linear_act(x, w, b, activation=act)
        rest = torch.ones(130, dtype=torch.bool)
        rest[1:4] = False
        want = act64(torch.tensor(0.5, dtype=torch.float64), act)[0].item()
        assert torch.allclose(y[rest].double().cpu(), torch.tensor(want).double(), rtol=2 ** -7)
        assert (y[1] == inf).all()
        assert (y[2] == (-inf if act is None else 0)).all()
        assert torch.isnan(y[3]).all()
        dx, = torch.autograd.grad(y, x, torch.ones_like(y))
        assert torch.isfinite(dx[rest]).all()
        assert (dx[1, 0] == 20).all() and (dx[2, 0] == (20 if act is None else 0)).all()
        assert torch.isnan(dx[3, 0]) or act is None


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("act", ["gelu", "gelu_tanh", "silu"])
def test_activation_over_its_range(act, dtype):
    """Through a unit weight, so z is exact: the value is off by its rounding and some 1e-6 of itself
    (2^-18, the exponential's relative error far out), the derivative by half a step of 2^-14 and
    2^-20, and by its rounding as dx."""
    from turboadam_b200 import linear_act

    x = torch.cat([torch.linspace(-s, s, 40001, device="cuda") for s in (1.0, 6.0, 40.0)])
    x = x.to(dtype).view(-1, 1).requires_grad_(True)
    w = torch.ones(8, 1, device="cuda", dtype=dtype)
    y = linear_act(x, w, activation=act)
    z = x.detach().double()
    v, d = act64(z, act)
    want = v.expand_as(y)
    u = U[dtype]
    within(y.detach(), want, (u + 2.0 ** -18) * want.abs() + 2.0 ** -21 * z.abs().clamp(max=1.0)
           + 2.0 ** -25, "y")
    dy = torch.zeros_like(y)
    dy[:, 3] = 1
    dx, = torch.autograd.grad(y, x, dy)
    within(dx, d, (2.0 ** -15 + 2.0 ** -20) * (1 + 4 * u) + 2 * u * d.abs() + 2.0 ** -25, "dx")


def test_linear_gradient_by_differences():
    """<grad, v> against a central difference of the layer itself, in every argument.

    fp16 outputs carry 2^-11 of |y| each, independent, so a sum of n of them weighted by dy is
    off by about 2^-11 |y||dy| / sqrt(3) (2-norms of the products); six times that over 2h, plus
    the cubic term h^2 / 6 times |act'''| <= 2 of |dz change|^3, bounds the difference."""
    from turboadam_b200 import linear_act

    h = 2.0 ** -4
    for act in ("gelu", "silu", "gelu_tanh"):
        c = make_linear(64, 48, 80, torch.float16, seed=5)
        args = [c[k].detach().requires_grad_(True) for k in "xwbr"]
        y = linear_act(args[0], args[1], args[2], act, args[3])
        grads = torch.autograd.grad(y, args, c["dy"])
        dy = c["dy"].double()
        gen = torch.Generator(device="cuda").manual_seed(9)
        for i, a in enumerate(args):
            v = torch.sign(torch.randn(a.shape, device="cuda", generator=gen)).half()
            if i == 1:
                v = v / 8
            outs, ends = [], []
            for sgn in (1, -1):
                moved = [t.detach() for t in args]
                moved[i] = (moved[i].double() + sgn * h * v.double()).half()
                ends.append(moved[i].double())
                outs.append(linear_act(moved[0], moved[1], moved[2], act, moved[3]).double())
            diff = (dy * (outs[0] - outs[1])).sum().item()
            step = ends[0] - ends[1]  # the difference really taken, after rounding
            want = (grads[i].double() * step).sum().item()
            noise = 6 * 2.0 ** -11 / math.sqrt(3) * 2 * (dy * outs[0]).norm().item()
            mid = [t.detach().double() for t in args]
            if i == 0:
                dz = step @ mid[1].t() / 2
            elif i == 1:
                dz = mid[0] @ step.t() / 2
            else:
                dz = (step / 2).expand(64, 80)
            cubic = 2 / 6 * 2 * (dy.abs() * dz.abs() ** 3).sum().item() if i < 3 else 0.0
            grad_err = 2.0 ** -10 * (grads[i].double().abs() * step.abs()).norm().item() * 6
            assert abs(diff - want) <= noise + cubic + grad_err, (act, i, diff, want)


def test_linear_offsets_past_32_bits():
    """An output of over 2^31 elements."""
    from turboadam_b200 import linear_act

    t, i, o = 66000, 16, 33000
    x = torch.randn(t, i, device="cuda").bfloat16()
    w = torch.randn(o, i, device="cuda").bfloat16()
    y = linear_act(x, w)
    rows = torch.tensor([0, 1, 65000, 65536, t - 1], device="cuda")
    want = x[rows].double() @ w.double().t()
    within(y[rows], want, 2.0 ** -8 * want.abs() + 1e-4, "y")


def test_linear_is_deterministic():
    from turboadam_b200 import linear_act

    for sizes in ((3, 4096, 100), (100, 4096, 200), (2048, 768, 2304)):
        c = make_linear(*sizes, torch.bfloat16)
        first = None
        for _ in range(3):
            x, w, b = (c[k].detach().requires_grad_(True) for k in "xwb")
            y = linear_act(x, w, b, activation="silu")
            out = [y, *torch.autograd.grad(y, (x, w, b), c["dy"])]
            first = first or out
            assert all(torch.equal(p, q) for p, q in zip(out, first))


def test_linear_refusals():
    from turboadam_b200 import linear_act

    x = torch.randn(4, 8, device="cuda").bfloat16()
    w = torch.randn(6, 8, device="cuda").bfloat16()
    with pytest.raises(NotImplementedError):
        linear_act(x.float(), w.float())
    for bad in (dict(weight=w.half()), dict(weight=w[:, :7]), dict(weight=w[0]),
                dict(weight=w, bias=x[0]), dict(weight=w, bias=w[:, 0].half()),
                dict(weight=w, activation="tanh"), dict(weight=w, residual=x),
                dict(weight=w.cpu()), dict(weight=w, residual=torch.zeros(4, 6, device="cuda"))):
        with pytest.raises(ValueError):
            linear_act(x, **bad)


# ---------------------------------------------------------------------------
def ortho64(x, steps=5, coefficients=QUINTIC, eps=1e-7):
    x = x.double()
    x = x / (x.square().sum((-2, -1), keepdim=True).sqrt() + eps)
    tall = x.shape[-2] > x.shape[-1]
    x = x.mT if tall else x
    rows = [coefficients] * steps if not hasattr(coefficients[0], "__len__") else coefficients
    for a, b, c in rows:
        g = x @ x.mT
        x = a * x + (b * g + c * (g @ g)) @ x
    return x.mT if tall else x


def rel(got, want):
    return ((got.double() - want).norm() / want.norm().clamp(min=1e-300)).item()


def grad_like(*shape, dtype=torch.float32, seed=0):
    """Gaussian noise under a few strong directions."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(*shape, device="cuda", generator=g) * 0.05
    r = max(1, min(shape[-2:]) // 4)
    u = torch.randn(*shape[:-1], r, device="cuda", generator=g)
    v = torch.randn(*shape[:-2], r, shape[-1], device="cuda", generator=g)
    s = torch.exp(-4.0 * torch.arange(r, device="cuda") / r) / math.sqrt(r)
    return ((x + (u * s) @ v) * 1e-3).to(dtype)


ORTHO_SHAPES = [(1, 1), (1, 7), (7, 1), (2, 3), (8, 8), (63, 65), (65, 63), (96, 70), (128, 128),
                (129, 127), (5, 64, 200), (3, 200, 64), (256, 256), (257, 300), (300, 257),
                (16, 3000), (3001, 17), (1000, 129), (12, 320, 320), (2, 3, 80, 72),
                (700, 1500), (1500, 700), (2, 1024, 1032), (2560, 2600)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32, torch.float16])
@pytest.mark.parametrize("shape", ORTHO_SHAPES)
def test_ortho_shapes(shape, dtype):
    from turboadam_b200 import orthogonalize

    x = grad_like(*shape)
    x = (x * 1e3).to(dtype) if dtype == torch.float16 else x.to(dtype)
    got = orthogonalize(x, dtype=torch.float32)
    assert got.shape == x.shape and rel(got, ortho64(x)) <= ORTHO_TOL
    low = orthogonalize(x)
    assert low.dtype == torch.bfloat16
    within(low, got.double(), 2.0 ** -8 * got.double().abs() + 1e-30, "bf16 result")


@pytest.mark.parametrize("steps", [1, 2, 3, 4, 7])
def test_ortho_steps(steps):
    from turboadam_b200 import orthogonalize

    for dtype in (torch.bfloat16, torch.float32):
        for shape in ((60, 90), (90, 60), (400, 900)):
            x = grad_like(*shape, dtype=dtype)
            got = orthogonalize(x, steps=steps, dtype=torch.float32)
            assert rel(got, ortho64(x, steps)) <= ORTHO_TOL * steps / 5 + 1e-3


def test_ortho_coefficients_per_step():
    """A cubic schedule that converges: the result has orthonormal rows."""
    from turboadam_b200 import orthogonalize

    x = torch.randn(64, 200, device="cuda")
    rows = [QUINTIC] * 4 + [(1.5, -0.5, 0.0)] * 6
    got = orthogonalize(x, steps=10, coefficients=rows, dtype=torch.float32)
    assert rel(got, ortho64(x, 10, rows)) <= 2 * ORTHO_TOL
    eye = torch.eye(64, device="cuda", dtype=torch.float64)
    assert rel(got.double() @ got.double().t(), eye) <= 2 * ORTHO_TOL
    # and it is the polar factor
    u, _, vh = torch.linalg.svd(x.double(), full_matrices=False)
    assert rel(got, u @ vh) <= 2 * ORTHO_TOL


@pytest.mark.parametrize("scale", [1e-30, 1e-12, 1.0, 1e12, 1e30])
def test_ortho_scales(scale):
    """The norm is taken in 64 bits: squares outside fp32's range do not matter (eps = 0)."""
    from turboadam_b200 import orthogonalize

    for shape in ((60, 90), (300, 200)):
        x = torch.randn(*shape, device="cuda") * scale
        got = orthogonalize(x, eps=0.0, dtype=torch.float32)
        assert rel(got, ortho64(x, eps=0.0)) <= ORTHO_TOL


def test_ortho_eps_matters_for_small_inputs():
    from turboadam_b200 import orthogonalize

    for shape in ((60, 90), (300, 200)):
        x = torch.randn(*shape, device="cuda") * 1e-9
        for eps in (1e-7, 1e-5):
            assert rel(orthogonalize(x, eps=eps, dtype=torch.float32),
                       ortho64(x, eps=eps)) <= ORTHO_TOL


def test_ortho_zero_and_non_finite_matrices_in_a_stack():
    from turboadam_b200 import orthogonalize

    for shape in ((6, 40, 60), (6, 60, 40), (6, 200, 264)):
        x = torch.randn(*shape, device="cuda")
        clean = orthogonalize(x, dtype=torch.float32)
        y = x.clone()
        y[1] = 0
        y[3, 2, 5] = float("nan")
        y[4, 0, 0] = float("inf")
        got = orthogonalize(y, dtype=torch.float32)
        assert (got[1] == 0).all()
        assert torch.isnan(got[3]).all() and torch.isnan(got[4]).all()
        for i in (0, 2, 5):
            assert torch.equal(got[i], clean[i])
        one = torch.zeros(*shape[1:], device="cuda")
        assert (orthogonalize(one, eps=0.0) == 0).all()


def test_ortho_rank_deficient():
    """Zero rows, repeated rows: singular values of zero stay near zero."""
    from turboadam_b200 import orthogonalize

    for shape in ((100, 140), (300, 500)):
        x = torch.randn(*shape, device="cuda").bfloat16()
        x[10:40] = 0
        x[50:60] = x[60:70]
        got = orthogonalize(x, dtype=torch.float32)
        assert (got[10:40] == 0).all()
        assert rel(got, ortho64(x)) <= ORTHO_TOL


def test_ortho_strided_unaligned_and_empty():
    from turboadam_b200 import orthogonalize

    base = torch.randn(130, 211, device="cuda")
    for x in (base[:, 1:98], base.t()[:100], base[::2], base.reshape(-1)[3:3 + 90 * 80].view(90, 80),
              base.bfloat16().reshape(-1)[1:1 + 90 * 80].view(90, 80)):
        assert rel(orthogonalize(x, dtype=torch.float32), ortho64(x)) <= ORTHO_TOL
    for shape in ((0, 5), (5, 0), (0, 5, 5), (2, 0, 3)):
        assert orthogonalize(torch.empty(*shape, device="cuda")).shape == shape


def test_ortho_offsets_past_32_bits():
    """A stack of over 2^31 elements; its last matrices are checked."""
    from turboadam_b200 import orthogonalize

    n = 2050
    x = torch.empty(n, 1024, 1024, device="cuda", dtype=torch.bfloat16).normal_()
    got = orthogonalize(x)
    for i in (0, 1023, n - 1):
        assert rel(got[i], ortho64(x[i])) <= ORTHO_TOL + 2.0 ** -8


def test_ortho_is_deterministic_and_stream_ordered():
    from turboadam_b200 import orthogonalize

    side = torch.cuda.Stream()
    for shape in ((96, 70), (300, 4000), (12, 256, 256)):
        x = torch.randn(*shape, device="cuda")
        first = orthogonalize(x)
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            y = x * 2  # made on the side stream
            outs = [orthogonalize(y) for _ in range(4)]
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(orthogonalize(x), first)
        # scaling by a power of two changes no bit but through eps (1e-7 of a norm over 50)
        assert all(torch.equal(o, outs[0]) for o in outs)
        assert rel(outs[0], first.double()) <= 1e-3


def test_ortho_graph_capture():
    from turboadam_b200 import orthogonalize

    for shape in ((96, 70), (3, 200, 300)):
        x = torch.randn(*shape, device="cuda")
        orthogonalize(x)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = orthogonalize(x)
        for seed in (1, 2):
            torch.manual_seed(seed)
            x.copy_(torch.randn(*shape, device="cuda"))
            g.replay()
            assert torch.equal(out, orthogonalize(x))
        del g


def test_ortho_refusals():
    from turboadam_b200 import orthogonalize

    x = torch.randn(4, 6, device="cuda")
    with pytest.raises(ValueError):
        orthogonalize(x[0])
    with pytest.raises(NotImplementedError):
        orthogonalize(x.double())
    with pytest.raises(NotImplementedError):
        orthogonalize(x, dtype=torch.float64)
    for kw in (dict(steps=0), dict(eps=-1.0), dict(coefficients=(1.0, 2.0)), dict(steps=33)):
        with pytest.raises(ValueError):
            orthogonalize(x, **kw)


# ---------------------------------------------------------------------------
def muon64(p, g, m, group):
    mu = group["momentum"]
    m = mu * m.double() + (1 - mu) * g.double()
    u = mu * m + (1 - mu) * g.double() if group["nesterov"] else m
    r, c = p.shape[-2:]
    if group["adjust_lr_fn"] == "match_rms_adamw":
        s = 0.2 * math.sqrt(max(r, c))
    else:
        s = math.sqrt(max(1.0, r / c))
    o = ortho64(u, group["ns_steps"], group["ns_coefficients"], group["eps"])
    return p.double() * (1 - group["lr"] * group["weight_decay"]), group["lr"] * s * o, m


MUON_SHAPES = [(96, 70), (300, 200), (50, 768), (1000, 129), (4, 64, 48), (300, 200), (1, 9),
               (512, 640), (33, 1), (2, 3, 40, 56)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("kw", [dict(), dict(nesterov=False, momentum=0.9),
                                dict(adjust_lr_fn="match_rms_adamw", ns_steps=3),
                                dict(momentum_dtype=torch.bfloat16, weight_decay=0.0)])
def test_muon_step(dtype, kw):
    from turboadam_b200 import Muon

    params = [torch.nn.Parameter((torch.randn(*s, device="cuda") * 0.02).to(dtype))
              for s in MUON_SHAPES]
    opt = Muon(params, lr=0.02, **kw)
    u_m = U[kw.get("momentum_dtype", torch.float32)]
    for step in range(3):
        for i, p in enumerate(params):
            p.grad = grad_like(*p.shape, seed=31 * step + i).mul(100).to(dtype)
        before = [(p.detach().clone(), opt.state[p].get("momentum_buffer",
                                                        torch.zeros_like(p)).clone())
                  for p in params]
        opt.step()
        for p, (p0, m0) in zip(params, before):
            keep, move, m = muon64(p0, p.grad, m0, opt.param_groups[0])
            got = opt.state[p]["momentum_buffer"]
            assert got.dtype == kw.get("momentum_dtype", torch.float32)
            within(got, m, (u_m + 2.0 ** -22) * (m.abs() + m0.double().abs() +
                                                 p.grad.double().abs()) + 1e-30, "momentum")
            # the direction is taken from the momentum as stored
            dm = 1.0 if u_m > 2.0 ** -20 else 0.0
            err = (p.detach().double() - (keep - move)).norm().item()
            tol = ((ORTHO_TOL + dm * 4 * u_m) * move.norm() +
                   (U[dtype] + 2.0 ** -22) * (keep.norm() + move.norm())).item()
            assert err <= tol, (tuple(p.shape), err, tol)


def test_muon_is_the_orthogonalised_update():
    """The fused update equals orthogonalize of the direction, up to its rounding."""
    from turboadam_b200 import Muon, orthogonalize

    p = torch.nn.Parameter(torch.zeros(300, 400, device="cuda"))
    p.grad = torch.randn(300, 400, device="cuda").bfloat16().float()
    Muon([p], lr=1.0, weight_decay=0.0, momentum=0.0, nesterov=False).step()
    o = orthogonalize(p.grad.bfloat16(), dtype=torch.float32)
    assert rel(-p.detach(), o.double()) <= 1e-6


def test_muon_lists_longer_than_a_launch():
    """More shapes than a launch holds, more matrices than a table launch holds, and a workspace
    limit that cuts the list."""
    from turboadam_b200 import Muon, muon

    shapes = [(16 + 7 * i, 90 - 5 * i) for i in range(11)] * 3
    gs = [grad_like(*s, seed=i) for i, s in enumerate(shapes)]

    def run():
        ps = [torch.nn.Parameter(torch.full(s, 0.5, device="cuda")) for s in shapes]
        opt = Muon(ps, lr=0.1)
        for p, g in zip(ps, gs):
            p.grad = g.clone()
        opt.step()
        return [p.detach() for p in ps]

    whole = run()
    limit = muon.WORKSPACE_LIMIT
    try:
        muon.WORKSPACE_LIMIT = 200_000
        parts = run()
    finally:
        muon.WORKSPACE_LIMIT = limit
    for a, b, g in zip(whole, parts, gs):
        assert torch.equal(a, b)
        keep, move, _ = muon64(torch.full_like(g, 0.5), g, torch.zeros_like(g),
                               dict(momentum=0.95, nesterov=True, adjust_lr_fn=None, ns_steps=5,
                                    ns_coefficients=QUINTIC, eps=1e-7, lr=0.1, weight_decay=0.1))
        assert ((a.double() - keep + move).norm() <= ORTHO_TOL * move.norm() + 1e-6 * keep.norm())


def test_muon_state_dict_round_trip():
    from turboadam_b200 import Muon

    def make(dtype):
        torch.manual_seed(3)
        return [torch.nn.Parameter(torch.randn(60, 80, device="cuda").to(dtype)),
                torch.nn.Parameter(torch.randn(2, 30, 20, device="cuda").to(dtype))]

    a = make(torch.bfloat16)
    opt = Muon(a, lr=0.05)
    for p in a:
        p.grad = torch.randn_like(p)
    opt.step()
    b = [torch.nn.Parameter(p.detach().clone()) for p in a]
    other = Muon(b, lr=0.05)
    other.load_state_dict(opt.state_dict())
    for p, q in zip(a, b):
        m = other.state[q]["momentum_buffer"]
        assert m.dtype == torch.float32 and torch.equal(m, opt.state[p]["momentum_buffer"])
        assert m.data_ptr() != opt.state[p]["momentum_buffer"].data_ptr()
        q.grad = p.grad.clone()
    opt.step()
    other.step()
    assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_muon_graph_capture():
    from turboadam_b200 import Muon

    def make():
        torch.manual_seed(7)
        ps = [torch.nn.Parameter(torch.randn(*s, device="cuda")) for s in ((64, 96), (300, 130))]
        for p in ps:
            p.grad = torch.randn_like(p)
        return ps, Muon(ps, lr=0.02)

    ps, opt = make()
    opt.step()  # the momentum exists before the capture
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        opt.step()
    g.replay()
    g.replay()
    torch.cuda.synchronize()
    qs, eager = make()
    for _ in range(3):
        eager.step()
    assert all(torch.equal(p, q) for p, q in zip(ps, qs))
    del g


def test_muon_skips_missing_gradients_and_refuses_others():
    from turboadam_b200 import Muon

    a = torch.nn.Parameter(torch.randn(30, 40, device="cuda"))
    b = torch.nn.Parameter(torch.randn(30, 40, device="cuda"))
    before = b.detach().clone()
    opt = Muon([a, b], lr=0.1)
    a.grad = torch.randn_like(a)
    assert opt.step(lambda: 3.5) == 3.5
    assert torch.equal(b, before) and b not in opt.state
    c = torch.nn.Parameter(torch.randn(30, 40, device="cuda").t())
    c.grad = torch.randn(40, 30, device="cuda")
    with pytest.raises(NotImplementedError, match="contiguous"):
        Muon([c]).step()
    d = torch.nn.Parameter(torch.randn(30, 40, device="cuda").double())
    d.grad = torch.randn_like(d)
    with pytest.raises(NotImplementedError):
        Muon([d]).step()


def test_muon_non_finite_gradient_stays_in_its_matrix():
    from turboadam_b200 import Muon

    ps = [torch.nn.Parameter(torch.randn(40, 60, device="cuda")) for _ in range(3)]
    for p in ps:
        p.grad = torch.randn_like(p)
    ps[1].grad[3, 4] = float("inf")
    Muon(ps).step()
    assert torch.isnan(ps[1]).all()
    assert torch.isfinite(ps[0]).all() and torch.isfinite(ps[2]).all()


# ---------------------------------------------------------------------------
@pytest.mark.parametrize("shape", [(2048, 4200), (4100, 2050)])
def test_ortho_steps_in_pairs(shape):
    """Sides from which the later steps also go in pairs."""
    from turboadam_b200 import orthogonalize

    for dtype in (torch.bfloat16, torch.float32):
        x = grad_like(*shape, dtype=dtype)
        assert rel(orthogonalize(x, dtype=torch.float32), ortho64(x)) <= ORTHO_TOL


def test_ortho_split_sums_and_mixed_lists():
    """A long sum over few tiles (split over SMs), beside shapes of both sequences of steps and
    both kinds of result, in one call of the optimizer."""
    from turboadam_b200 import Muon

    shapes = [(40, 9000), (9000, 24), (2048, 4100), (130, 130), (40, 9000)]
    for dtype in (torch.float32, torch.bfloat16):
        ps = [torch.nn.Parameter(torch.zeros(s, device="cuda", dtype=dtype)) for s in shapes]
        opt = Muon(ps, lr=1.0, weight_decay=0.0, momentum=0.0, nesterov=False)
        for i, p in enumerate(ps):
            p.grad = grad_like(*p.shape, seed=i).to(dtype)
        opt.step()
        for p in ps:
            want = ortho64(p.grad) * math.sqrt(max(1.0, p.shape[0] / p.shape[1]))
            tol = ORTHO_TOL + (2.0 ** -8 if dtype == torch.bfloat16 else 0.0)
            assert rel(-p.detach(), want) <= tol


def test_residual_mlp_example_learns():
    """The layers, the orthogonal start and both optimizers together: the loss falls by far."""
    import importlib.util
    import os

    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples",
                        "train_residual_mlp.py")
    spec = importlib.util.spec_from_file_location("train_residual_mlp", path)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    losses = example.train(steps=120, width=128, depth=2, batch=256)
    assert all(math.isfinite(v) for v in losses)
    assert sum(losses[-10:]) < 0.2 * sum(losses[:10])


def test_operators_on_two_streams_at_once():
    """Independent calls on two streams: each chain's blocks are resident together whatever else
    runs, and workspaces are not shared."""
    from turboadam_b200 import linear_act, orthogonalize

    xs = [torch.randn(12, 256, 320, device="cuda"), torch.randn(40, 100, 90, device="cuda")]
    w = torch.randn(512, 320, device="cuda").bfloat16()
    t = torch.randn(900, 320, device="cuda").bfloat16()
    want = [orthogonalize(x) for x in xs] + [linear_act(t, w, activation="silu")]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append((orthogonalize(xs[i]), linear_act(t, w, activation="silu")))
    torch.cuda.synchronize()
    for i in range(2):
        for o, y in got[i]:
            assert torch.equal(o, want[i]) and torch.equal(y, want[2])
