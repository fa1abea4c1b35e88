"""The matrix operators beside the packed optimizer step, as cases to time and compare.

Three operators, which a weight matrix meets in this order in a training step: the fused linear
layer and its gradients (``linear_act``), the orthogonalisation of an update by Newton-Schulz
products (``orthogonalize``), and the optimizer step built on it (``Muon``). ``run`` computes a
case in its plain form (elementary torch operations in 32 bits, rounded once at the end) or, where
``own`` is true, through the package; ``exact`` gives the definition's values in 64 bits.
"""
import math

import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
# the quintic of the Muon optimizer: X <- aX + bAX + cA^2X with A = XX^T, five times
COEFFS, STEPS, EPS = (3.4445, -4.7750, 2.0315), 5, 1e-7
# an ordinary Muon setting
HYPER = dict(lr=0.02, momentum=0.95, weight_decay=0.1)


def listed():
    return [
        # one small adapter-sized matrix, odd in both sizes: latency counts
        dict(name="ortho one 96x70", op="ortho", batch=1, rows=96, cols=70, dtype="fp32"),
        # the attention output projections of all 12 layers of a GPT-2-small
        dict(name="ortho gpt2 12x768x768", op="ortho", batch=12, rows=768, cols=768, dtype="bf16"),
        # ragged in both sizes, fp32 gradients
        dict(name="ortho ragged 1000x4099", op="ortho", batch=1, rows=1000, cols=4099,
             dtype="fp32"),
        # a Llama-3-8B key projection: few output tiles, a long sum
        dict(name="ortho kv 1024x4096", op="ortho", batch=1, rows=1024, cols=4096, dtype="bf16"),
        # a Llama-3-8B gate projection: tall, bound by the products
        dict(name="ortho gate 14336x4096", op="ortho", batch=1, rows=14336, cols=4096,
             dtype="bf16"),
        # a step over a small model's odd matrices: latency counts
        dict(name="muon small odd", op="muon", shapes="300x200 96x70 50x768 1000x129",
             dtype="bf16"),
        # a step over the attention matrices of 4 GPT-2-small layers
        dict(name="muon gpt2 attention x4", op="muon", shapes=" ".join(["768x2304 768x768"] * 4),
             dtype="bf16"),
        # a step over one Llama-3-8B layer (q k v o gate up down)
        dict(name="muon llama layer", op="muon", dtype="bf16",
             shapes="4096x4096 1024x4096 1024x4096 4096x4096 14336x4096 14336x4096 4096x14336"),
        # serving: one token through a Llama-3-8B gate projection, bound by the weight's bytes
        dict(name="linear token 4096>14336", op="linear", tokens=1, fan_in=4096, fan_out=14336,
             dtype="bf16", act="silu", bias=False, residual=False, layout="oi", train=False),
        # training: GPT-2-small's fused qkv layer (stored input by output), 8 x 1024 tokens
        dict(name="linear gpt2 8192 768>2304", op="linear", tokens=8192, fan_in=768,
             fan_out=2304, dtype="bf16", act="none", bias=True, residual=False, layout="io",
             train=True),
        # training: Llama-3-8B's gate layer on 8192 tokens, bound by the products
        dict(name="linear gate 8192 4096>14336", op="linear", tokens=8192, fan_in=4096,
             fan_out=14336, dtype="bf16", act="silu", bias=False, residual=False, layout="oi",
             train=True),
        # odd in every size, fp16, with every part of the epilogue
        dict(name="linear odd 777 1001>1003", op="linear", tokens=777, fan_in=1001, fan_out=1003,
             dtype="fp16", act="gelu", bias=True, residual=True, layout="oi", train=True),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(["ortho", "muon", "linear"])
    if op == "ortho":
        rows, cols = _log(rng, 16, 8192), _log(rng, 16, 8192)
        room = 14336 * 4096 * 4096 // (rows * cols * min(rows, cols))
        return dict(op=op, batch=_log(rng, 1, max(1, min(16, room))), rows=rows, cols=cols,
                    dtype=rng.choice(["bf16", "fp32"]))
    if op == "muon":
        shapes = ["%dx%d" % (_log(rng, 16, 4096), _log(rng, 16, 4096))
                  for _ in range(rng.randint(1, 8))]
        return dict(op=op, shapes=" ".join(shapes), dtype="bf16")
    tokens, fan_in = _log(rng, 1, 16384), _log(rng, 16, 16384)
    fan_out = min(_log(rng, 16, 16384), max(16, 8192 * 4096 * 14336 // (tokens * fan_in)))
    return dict(op=op, tokens=tokens, fan_in=fan_in, fan_out=fan_out,
                dtype=rng.choice(["bf16", "fp16"]),
                act=rng.choice(["none", "relu", "gelu", "silu"]),
                bias=rng.random() < 0.5, residual=rng.random() < 0.5,
                layout=rng.choice(["oi", "io"]), train=rng.random() < 0.6)


def _shapes(case):
    return [tuple(int(v) for v in s.split("x")) for s in case["shapes"].split()]


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _gradient(gen, batch, rows, cols, dtype):
    """A weight gradient's spectrum: a few strong directions, which decay, over a noise floor."""
    rank = max(1, min(rows, cols, 256) // 4)
    s = torch.exp(-4.0 * torch.arange(rank, device=DEV) / rank) / math.sqrt(rank)
    left = torch.randn(batch, rows, rank, device=DEV, generator=gen) * s
    right = torch.randn(batch, rank, cols, device=DEV, generator=gen)
    g = torch.randn(batch, rows, cols, device=DEV, generator=gen).mul_(0.05)
    return g.baddbmm_(left, right).mul_(1e-3).to(dtype)


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    if case["op"] == "ortho":
        g = _gradient(gen, case["batch"], case["rows"], case["cols"], dtype)
        return dict(case=case, x=g)
    if case["op"] == "muon":
        st = dict(case=case, params=[], grads=[], momentum=[])
        for rows, cols in _shapes(case):
            p = torch.randn(rows, cols, device=DEV, generator=gen).mul_(0.02)
            st["params"].append(p.to(dtype))
            st["grads"].append(_gradient(gen, 1, rows, cols, dtype)[0])
            st["momentum"].append(_gradient(gen, 1, rows, cols, torch.float32)[0])
        if own:  # the optimizer a training program holds, resumed with its momentum
            from turboadam_b200 import Muon

            for p, g in zip(st["params"], st["grads"]):
                p.grad = g
            st["opt"] = Muon(st["params"], **HYPER)
            for p, m in zip(st["params"], st["momentum"]):
                st["opt"].state[p]["momentum_buffer"] = m
        return st
    t, i, o = case["tokens"], case["fan_in"], case["fan_out"]
    w = torch.randn((o, i) if case["layout"] == "oi" else (i, o), device=DEV, generator=gen)
    w = w.mul_(1.0 / math.sqrt(i)).to(dtype)
    st = dict(case=case, w=w if case["layout"] == "oi" else w.t(),
              x=torch.randn(t, i, device=DEV, generator=gen).to(dtype), b=None, r=None, dy=None)
    if case["bias"]:
        st["b"] = torch.randn(o, device=DEV, generator=gen).mul_(0.1).to(dtype)
    if case["residual"]:
        st["r"] = torch.randn(t, o, device=DEV, generator=gen).to(dtype)
    if case["train"]:
        st["dy"] = torch.randn(t, o, device=DEV, generator=gen).to(dtype)
        for k in "xwbr":
            if st[k] is not None:
                st[k].requires_grad_(True)
    return st


# ---------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------
def _newton_schulz(x):
    x = x.float()
    tall = x.shape[-2] > x.shape[-1]
    if tall:
        x = x.mT
    x = x / (x.square().sum((-2, -1), keepdim=True).sqrt() + EPS)
    a, b, c = COEFFS
    for _ in range(STEPS):
        gram = x @ x.mT
        x = a * x + (b * gram + c * (gram @ gram)) @ x
    return x.mT if tall else x


def _muon_plain(st):
    lr, mu, wd = HYPER["lr"], HYPER["momentum"], HYPER["weight_decay"]
    for p, g, m in zip(st["params"], st["grads"], st["momentum"]):
        g = g.float()
        m.mul_(mu).add_(g, alpha=1 - mu)
        o = _newton_schulz((1 - mu) * g + mu * m)
        scale = math.sqrt(max(1.0, p.shape[0] / p.shape[1]))
        p.copy_(p.float() * (1 - lr * wd) - lr * scale * o)
    return dict(params=st["params"], momentum=st["momentum"])


def _act(z, kind):
    """The activation and its derivative."""
    if kind == "relu":
        return z.clamp(min=0), (z > 0).to(z.dtype)
    if kind == "gelu":
        cdf = 0.5 * (1 + torch.erf(z * math.sqrt(0.5)))
        return z * cdf, cdf + z * torch.exp(-0.5 * z * z) * (1 / math.sqrt(2 * math.pi))
    if kind == "silu":
        s = 1 / (1 + torch.exp(-z))
        return z * s, s * (1 + z * (1 - s))
    return z, torch.ones_like(z)


def _linear(st, to):
    """y = act(x w^T + b) + r and, in training, the gradients of sum(y dy)."""
    case, dtype = st["case"], st["x"].dtype
    x, w = st["x"].detach().to(to), st["w"].detach().to(to)
    z = x @ w.t()
    if st["b"] is not None:
        z = z + st["b"].detach().to(to)
    y, d = _act(z, case["act"])
    if st["r"] is not None:
        y = y + st["r"].detach().to(to)
    out = [y]
    if case["train"]:
        dz = st["dy"].to(to) * d
        out += [dz @ w, dz.t() @ x]
        if st["b"] is not None:
            out.append(dz.sum(0))
        if st["r"] is not None:
            out.append(st["dy"].to(to))
    return [v.to(dtype) for v in out] if to == torch.float32 else out


def run(st):
    op = st["case"]["op"]
    if not own:
        if op == "ortho":
            return _newton_schulz(st["x"]).to(torch.bfloat16)
        return _muon_plain(st) if op == "muon" else _linear(st, torch.float32)
    import turboadam_b200 as ta

    if op == "ortho":
        return ta.orthogonalize(st["x"], steps=STEPS, coefficients=COEFFS, eps=EPS)
    if op == "muon":
        st["opt"].step()
        return dict(params=st["params"], momentum=st["momentum"])
    act = None if st["case"]["act"] == "none" else st["case"]["act"]
    y = ta.linear_act(st["x"], st["w"], st["b"], activation=act, residual=st["r"])
    if not st["case"]["train"]:
        return [y]
    leaves = [st[k] for k in "xwbr" if st[k] is not None]
    return [y.detach(), *torch.autograd.grad(y, leaves, st["dy"])]


# ---------------------------------------------------------------------------
# 64-bit values, from the definitions
# ---------------------------------------------------------------------------
def _polar64(x):
    """The iteration on a 64-bit matrix, by its action P_k ... P_1 on the normalised input with
    the smaller Gram matrix."""
    x = x.double()
    x = x / (torch.linalg.vector_norm(x) + EPS)
    a, b, c = COEFFS
    left = x.shape[0] <= x.shape[1]
    eye = torch.eye(min(x.shape), dtype=torch.float64, device=x.device)
    for _ in range(STEPS):
        g = torch.mm(x, x.t()) if left else torch.mm(x.t(), x)
        poly = torch.addmm(a * eye, g, b * eye + c * g)
        x = torch.mm(poly, x) if left else torch.mm(x, poly)
    return x


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "ortho":
        return torch.stack([_polar64(m) for m in st["x"]])
    if case["op"] == "linear":
        x, w = st["x"].detach().double(), st["w"].detach().double()
        z = torch.einsum("ti,oi->to", x, w)
        z = z if st["b"] is None else z + st["b"].detach().double()
        phi = {"none": lambda v: v, "relu": torch.relu, "silu": torch.nn.functional.silu,
               "gelu": torch.nn.functional.gelu}[case["act"]]
        if not case["train"]:
            y = phi(z)
            return [y if st["r"] is None else y + st["r"].detach().double()]
        z.requires_grad_(True)
        y = phi(z)
        dy = st["dy"].double()
        dz, = torch.autograd.grad(y, z, dy)
        y = y.detach()
        out = [y if st["r"] is None else y + st["r"].detach().double(),
               torch.einsum("to,oi->ti", dz, w), torch.einsum("to,ti->oi", dz, x)]
        if st["b"] is not None:
            out.append(torch.einsum("to->o", dz))
        if st["r"] is not None:
            out.append(dy)
        return out
    params, momentum = [], []
    mu = HYPER["momentum"]
    for p, g, m in zip(st["params"], st["grads"], st["momentum"]):
        m1 = m.double() + (1 - mu) * (g.double() - m.double())
        step = _polar64(g.double() + mu * (m1 - g.double()))
        r, c = p.shape
        gain = HYPER["lr"] * max(1.0, r / c) ** 0.5
        keep = 1 - HYPER["lr"] * HYPER["weight_decay"]
        params.append(torch.sub(p.double() * keep, step, alpha=gain))
        momentum.append(m1)
    return dict(params=params, momentum=momentum)


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------
def _polar_flops(rows, cols):
    """Per step X X^T and its square, symmetric (half of each), and the product with X."""
    s, t = min(rows, cols), max(rows, cols)
    return STEPS * (s * s * t + s ** 3 + 2 * s * s * t)


def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "ortho":
        n = case["batch"] * case["rows"] * case["cols"]
        return dict(bytes=n * (size + 2),
                    flops=case["batch"] * _polar_flops(case["rows"], case["cols"]))
    if case["op"] == "muon":
        # gradient read; parameter and momentum read and written
        return dict(bytes=sum(r * c * (3 * size + 8) for r, c in _shapes(case)),
                    flops=sum(_polar_flops(r, c) for r, c in _shapes(case)))
    t, i, o = case["tokens"], case["fan_in"], case["fan_out"]
    n = t * i + i * o + t * o + (o if case["bias"] else 0) + (t * o if case["residual"] else 0)
    if case["train"]:  # dy read; dx, dw, db and the residual's gradient (dy itself) returned
        n += t * o + t * i + i * o + (o if case["bias"] else 0)
    return dict(bytes=n * size, flops=(6 if case["train"] else 2) * t * i * o)
