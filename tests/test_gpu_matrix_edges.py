"""More edges of the matrix operators on the GPU: chains in which most SM pairs have no tile, and
what else the size lists of test_gpu_matrix.py do not reach. Bounds as derived there."""
import math

import pytest
import torch

from test_gpu_matrix import ORTHO_TOL, U, check_linear, make_linear, ortho64, rel, within

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _status_clean():
    from turboadam_b200 import matrix

    yield
    assert matrix.read_status() == 0


# ---------------------------------------------------------------------------
def test_ortho_pairs_without_tiles():
    """Phases of one size of tile list beside phases of another: in a 300 x 9000 matrix the Gram
    matrix's split sum occupies many pairs and its square two, so the other pairs pass a phase with
    nothing to do and take part in the next. Other work on the GPU shifts their warps against each
    other; every repetition gives the same bits and no wait runs out."""
    from turboadam_b200 import orthogonalize

    side = torch.cuda.Stream()
    noise = torch.randn(1 << 24, device="cuda")
    for shape in ((300, 9000), (9000, 300), (64, 20000), (2, 260, 3000)):
        x = torch.randn(*shape, device="cuda")
        first = orthogonalize(x, dtype=torch.float32)
        assert rel(first, ortho64(x)) <= ORTHO_TOL
        torch.cuda.synchronize()
        for i in range(30):
            with torch.cuda.stream(side):
                noise.mul_(1.0)
            assert torch.equal(orthogonalize(x, dtype=torch.float32), first)


# ---------------------------------------------------------------------------
@pytest.mark.parametrize("act", [None, "gelu", "relu"])
@pytest.mark.parametrize("layout", ["oi", "io"])
@pytest.mark.parametrize("tokens,fan_in", [(2, 8), (4, 768), (9, 768), (64, 768), (300, 8),
                                           (300, 65), (1, 768)])
def test_linear_one_output(tokens, fan_in, layout, act):
    """A value or reward head: its weight's gradient is a product whose left operand has one row,
    of elements that do not lie next to each other."""
    for dtype in (torch.bfloat16, torch.float16):
        check_linear(make_linear(tokens, fan_in, 1, dtype, layout), act)


def test_linear_one_input():
    """One input, the weight input by output: the weight's gradient has one row of x, here a column
    of a wider matrix."""
    for step, at in ((8, 0), (8, 2), (9, 2)):
        c = make_linear(40, 1, 64, torch.bfloat16)
        c["w"] = c["w"].reshape(1, 64).t()
        assert c["w"].stride() == (1, 64)
        wide = torch.randn(40, step, device="cuda").bfloat16()
        wide[:, at:at + 1] = c["x"]
        c["x"] = wide[:, at:at + 1]
        check_linear(c, "silu")


@pytest.mark.parametrize("fan_out", [64, 7])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_linear_one_strided_token(dtype, fan_out):
    """One token whose elements lie apart (a matrix's column, every other element), with and without
    copies of it, against weights of both layouts."""
    from turboadam_b200 import linear_act

    g = torch.Generator(device="cuda").manual_seed(3)
    m = torch.randn(96, 24, device="cuda", generator=g).to(dtype)
    odd = torch.randn(96, 25, device="cuda", generator=g).to(dtype)
    flat = torch.randn(1, 192, device="cuda", generator=g).to(dtype)
    tokens = (m[:, 3], m[:, 8], m[:, 3:4].t(), m[:, 16:17].t(), odd[:, 5], odd.t()[:1],
              flat[:, ::2], flat[0, 1::2])
    for w in (torch.randn(fan_out, 96, device="cuda", generator=g).to(dtype),
              torch.randn(96, fan_out, device="cuda", generator=g).to(dtype).t()):
        for x in tokens:
            y = linear_act(x, w)
            want = x.double() @ w.double().t()
            mag = x.double().abs() @ w.double().abs().t()
            assert y.shape == want.shape
            within(y, want, U[dtype] * want.abs() + 112 * 2.0 ** -22 * mag + 1e-6, "y")


# ---------------------------------------------------------------------------
@pytest.mark.parametrize("shape", [(1, 9), (60, 90), (90, 60), (300, 500), (500, 300), (3, 40, 64),
                                   (2, 520, 400), (1030, 1100)])
def test_ortho_float32_input_is_a_pair(shape):
    """One step with coefficients (1, 0, 0) returns X itself. A pair of fp16 numbers holds it to
    2^-22, the sums may truncate at 2^-22 and three roundings to fp32 follow: 2^-20 covers them;
    one fp16 number would leave some 2^-13."""
    from turboadam_b200 import orthogonalize

    x = torch.randn(*shape, device="cuda")
    got = orthogonalize(x, steps=1, coefficients=(1.0, 0.0, 0.0), dtype=torch.float32)
    want = x.double() / (x.double().square().sum((-2, -1), keepdim=True).sqrt() + 1e-7)
    assert rel(got, want) <= 2.0 ** -20


@pytest.mark.parametrize("shape", [(600, 700), (700, 600), (320, 640), (1024, 1280), (1280, 520)])
def test_ortho_low_half_of_a_pair(shape):
    """What the low half of a 32-bit input adds: with coefficients (0, 1, 0) one step is A X, and
    for x = hi + lo (hi an fp16 number, lo = +- 2^-12 hi by column, so that <hi, lo> = 0 and the
    norm stays) the difference to hi's result is A lo.

    A is rounded to fp16 (2^-11). The fp32 sums run over some K / 8 additions of truncated 2^-22
    each, of a sum 2^12 times the difference: at most K 2^-13, 0.13 at K = 1024, where every one is an
    error of full size and one sign, and a small part of that otherwise.
    (Blocks of A read the wrong way round would leave 0.3 and more.)"""
    from turboadam_b200 import orthogonalize

    rows, cols = sorted(shape)
    tall = shape[0] > shape[1]
    for seed in range(100):
        g = torch.Generator(device="cuda").manual_seed(seed)
        half = (torch.randn(rows, 3, device="cuda", generator=g) @
                torch.randn(3, cols // 2, device="cuda", generator=g))
        hi = torch.cat([half, half], 1).bfloat16().double()
        sign = torch.ones(cols, device="cuda", dtype=torch.float64)
        sign[cols // 2:] = -1
        lo = hi * sign * 2.0 ** -12
        # the scale that enters in fp32 has to be one number for both
        norms = torch.stack([hi.norm(), (hi + lo).norm()]) + 1e-7
        scales = (1.0 / norms).float()
        if scales[0] == scales[1]:
            break
    x = (hi + lo).float()
    assert torch.equal(x.double(), hi + lo)

    def step(m):
        m = m.float().t().contiguous() if tall else m.float()
        out = orthogonalize(m, steps=1, coefficients=(0.0, 1.0, 0.0), dtype=torch.float32)
        return (out.t() if tall else out).double()

    a = hi / norms[0]
    assert rel(step(x) - step(hi), (a @ a.t()) @ (lo / norms[0])) <= 0.1


# ---------------------------------------------------------------------------
def deriv64(z, act):
    """act' without cancellation far out on the negative side."""
    if act == "gelu":
        return (0.5 * torch.special.erfc(-z / math.sqrt(2)) +
                z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi))
    if act == "silu":
        s = torch.sigmoid(z)
        return s + z * s * torch.sigmoid(-z)
    k = 2 * math.sqrt(2 / math.pi)  # gelu_tanh: z sigmoid(k (z + 0.044715 z^3))
    w = k * (z + 0.044715 * z ** 3)
    s = torch.sigmoid(w)
    return s + z * s * torch.sigmoid(-w) * k * (1 + 3 * 0.044715 * z * z)


# what the derivative is kept to, relative: half the operand type's rounding; down to what size
KEPT = {torch.bfloat16: (2.0 ** -9, 2.0 ** -90), torch.float16: (2.0 ** -12, 2.0 ** -13)}


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("act,low", [("gelu", -10.0), ("gelu_tanh", -9.0), ("silu", -60.0)])
def test_linear_small_derivatives(act, low, dtype):
    """Far out on the negative side act' is small, and the gradient is as exact, relative to it, as
    elsewhere: its own error (2^-14: exponentials of arguments up to 75, themselves rounded), the
    code it is kept in, and the two roundings of dz and dx."""
    from turboadam_b200 import linear_act

    z = torch.cat([torch.linspace(low, -2.5, 30001), torch.linspace(-4.5, -2.5, 3001)])
    z = z.to(dtype).cuda().view(-1, 1)
    d = deriv64(z.double(), act)
    kept, least = KEPT[dtype]
    z, d = z[d.abs() >= least].view(-1, 1), d[d.abs() >= least].view(-1, 1)
    x = z.requires_grad_(True)
    w = torch.ones(8, 1, device="cuda", dtype=dtype)
    y = linear_act(x, w, activation=act)
    dy = torch.zeros_like(y)
    dy[:, 5] = 1
    dx, = torch.autograd.grad(y, x, dy)
    tiny = 2.0 ** -24 if dtype == torch.float16 else 0.0  # two roundings of a subnormal
    within(dx, d, (2 * U[dtype] + kept + 2.0 ** -14) * (1 + 4 * U[dtype]) * d.abs() + tiny, "dx")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("act,bias", [("gelu", -4.0), ("gelu_tanh", -4.0), ("silu", -10.0)])
@pytest.mark.parametrize("tokens", [1, 3, 200])
def test_linear_gradients_of_units_far_off(tokens, act, bias, dtype):
    """Units whose argument stays strongly negative: their bias and weight gradients relative to the
    sums of their terms' magnitudes. z is off by (K + 16) 2^-22 of its terms and act'' / act' is at
    most |z| + 2 there."""
    from turboadam_b200 import linear_act

    g = torch.Generator(device="cuda").manual_seed(tokens)
    x = (torch.randn(tokens, 16, device="cuda", generator=g) * 0.25).to(dtype)
    w = (torch.randn(24, 16, device="cuda", generator=g) * 0.05).to(dtype)
    b = torch.full((24,), bias, device="cuda", dtype=dtype)
    dy = (torch.rand(tokens, 24, device="cuda", generator=g) + 0.5).to(dtype)
    w.requires_grad_(True)
    b.requires_grad_(True)
    y = linear_act(x, w, b, activation=act)
    dw, db = torch.autograd.grad(y, (w, b), dy)
    xd, wd = x.double(), w.detach().double()
    z = xd @ wd.t() + bias
    z_err = 32 * 2.0 ** -22 * (xd.abs() @ wd.t().abs() + abs(bias))
    dz = dy.double() * deriv64(z, act)
    u = U[dtype]
    off = dz.abs() * (KEPT[dtype][0] + 2.0 ** -14 + (z.abs() + 2) * z_err)
    want = dz.sum(0)
    within(db, want, (off.sum(0) + (tokens + 16) * 2.0 ** -23 * dz.abs().sum(0)) * (1 + u) +
           u * want.abs() + 2.0 ** -25, "db")
    off = off + u * dz.abs() + 2.0 ** -25 * (dtype == torch.float16)
    want = dz.t() @ xd
    mag = dz.abs().t() @ xd.abs()
    within(dw, want, (off.t() @ xd.abs() + (tokens + 16) * 2.0 ** -22 * mag) * (1 + u) +
           u * want.abs() + 2.0 ** -25, "dw")


@pytest.mark.parametrize("act", ["relu", "gelu", "gelu_tanh", "silu"])
@pytest.mark.parametrize("tokens", [2, 40])
def test_linear_gradients_at_nan(tokens, act):
    """A NaN argument gives NaN gradients for its token and its unit's bias, and nothing else."""
    from turboadam_b200 import linear_act

    for dtype in (torch.bfloat16, torch.float16):
        x = torch.zeros(tokens, 16, device="cuda", dtype=dtype)
        x[1, 0] = float("nan")
        x.requires_grad_(True)
        w = torch.ones(8, 16, device="cuda", dtype=dtype)
        b = torch.zeros(8, device="cuda", dtype=dtype, requires_grad=True)
        y = linear_act(x, w, b, activation=act)
        dx, db = torch.autograd.grad(y, (x, b), torch.ones_like(y))
        assert torch.isnan(dx[1]).all() and torch.isnan(db).all()
        assert torch.isfinite(dx[0]).all() and torch.isfinite(dx[2:]).all()


# ---------------------------------------------------------------------------
def test_forward_mode_is_refused():
    """A tangent must not be lost without a word, in any argument."""
    from turboadam_b200 import linear_act, orthogonalize
    import torch.autograd.forward_ad as fwd

    bf = dict(device="cuda", dtype=torch.bfloat16)
    args = dict(x=torch.randn(4, 16, **bf), weight=torch.randn(8, 16, **bf),
                bias=torch.randn(8, **bf), residual=torch.randn(4, 8, **bf))
    for name in args:
        for grad in (False, True):
            with fwd.dual_level():
                dual = fwd.make_dual(args[name], torch.ones_like(args[name]))
                other = "x" if name != "x" else "weight"
                kw = {**args, name: dual, other: args[other].clone().requires_grad_(grad)}
                with pytest.raises(NotImplementedError, match="forward"):
                    linear_act(**kw)
    with fwd.dual_level():
        m = torch.randn(6, 9, device="cuda")
        with pytest.raises(NotImplementedError):
            orthogonalize(fwd.make_dual(m, torch.ones_like(m)))
        # without a tangent both run as ever
        assert orthogonalize(m).shape == (6, 9)
        assert linear_act(**args).shape == (4, 8)


def test_function_transforms_are_loud():
    """torch.func's transforms hand over tensors without storage."""
    from turboadam_b200 import linear_act, orthogonalize

    x = torch.randn(3, 4, 16, device="cuda").bfloat16()
    w = torch.randn(8, 16, device="cuda").bfloat16()
    with pytest.raises(RuntimeError):
        torch.func.vmap(lambda t: linear_act(t, w))(x)
    with pytest.raises((RuntimeError, NotImplementedError)):
        torch.func.jvp(lambda t: linear_act(t, w), (x,), (x,))
    with pytest.raises(RuntimeError):
        torch.func.vmap(orthogonalize)(x)
    with pytest.raises((RuntimeError, NotImplementedError)):
        torch.func.jvp(orthogonalize, (x,), (x,))
    with pytest.raises(RuntimeError):
        torch.func.grad(lambda t: linear_act(t, w).float().sum())(x)


# ---------------------------------------------------------------------------
def test_void_results_are_reported_by_the_next_call():
    """A wait that runs out (here the library's self-test, on the operators' own status word: a
    kernel whose copies never come, for 1 ms) makes the following calls raise until the status has
    been read, without a synchronisation of theirs."""
    from turboadam_b200 import Muon, _lib, linear_act, matrix, orthogonalize

    x = torch.randn(40, 16, device="cuda").bfloat16()
    w = torch.randn(8, 16, device="cuda").bfloat16()
    p = torch.nn.Parameter(torch.randn(16, 24, device="cuda"))
    p.grad = torch.randn_like(p)
    opt = Muon([p])
    opt.step()
    before = p.detach().clone()
    y = linear_act(x, w)
    out = torch.zeros(2, dtype=torch.int64, device="cuda")
    index = torch.cuda.current_device()
    lib = _lib.load()
    _lib.check(lib.ta_selftest_wait_timeout(1_000_000, matrix._word(index), out.data_ptr(),
                                            _lib.stream_ptr(index)), "self-test")
    torch.cuda.synchronize()
    for call in (lambda: linear_act(x, w), lambda: orthogonalize(p.detach()), opt.step):
        for _ in range(2):
            with pytest.raises(_lib.TurboAdamBackendError, match="void"):
                call()
    assert torch.equal(p.detach(), before)
    assert matrix.read_status(clear=False) == _lib.TA_STATUS_WAIT_TIMEOUT
    assert matrix.read_status() == _lib.TA_STATUS_WAIT_TIMEOUT
    assert matrix.read_status() == 0
    assert torch.equal(linear_act(x, w), y)
