"""Muon on B200: momentum, Newton-Schulz orthogonalisation and the decoupled
update of every weight matrix of a model in one call.

The matrices of a transformer go to :class:`Muon`, its vectors and embeddings
to :class:`turboadam_b200.TurboAdam`. The constructor's arguments, defaults and
state key follow ``torch.optim.Muon``; matrices may also be stacked ([...,
rows, cols], as the weights of a list of experts are).
"""
from __future__ import annotations

import math

import torch
from torch.optim import Optimizer

from . import _lib
from .matrix import _DTYPES, NS_COEFFICIENTS, NS_EPS, NS_STEPS, ortho_options, run_ortho

# workspace one call may take before the list is stepped in parts
WORKSPACE_LIMIT = 4 << 30


def _check_adjustment(kind):
    if kind not in (None, "original", "match_rms_adamw"):
        raise ValueError(f"adjust_lr_fn must be 'original' or 'match_rms_adamw', got {kind!r}")


def _gain(kind, lr, rows, cols):
    if kind == "match_rms_adamw":
        return lr * 0.2 * math.sqrt(max(rows, cols))
    return lr * math.sqrt(max(1.0, rows / cols))


def _check_group(group):
    lr, momentum, decay = group["lr"], group["momentum"], group["weight_decay"]
    if not lr >= 0:
        raise ValueError(f"lr must not be negative, got {lr}")
    if not 0 <= momentum < 1:
        raise ValueError(f"momentum must be in [0, 1), got {momentum}")
    if not decay >= 0:
        raise ValueError(f"weight_decay must not be negative, got {decay}")
    _check_adjustment(group["adjust_lr_fn"])
    ortho_options(group["ns_coefficients"], group["ns_steps"], group["eps"])  # checks them


class Muon(Optimizer):
    """Momentum orthogonalised by Newton-Schulz products.

    Per matrix, in one call for all of them: m <- momentum m + (1 - momentum) g;
    u = momentum m + (1 - momentum) g with ``nesterov``, else m; O = the
    Newton-Schulz iterate of u (:func:`turboadam_b200.orthogonalize`);
    p <- (1 - lr weight_decay) p - lr s O. ``adjust_lr_fn`` sets s:
    "original" (default) sqrt(max(1, rows / cols)), "match_rms_adamw"
    0.2 sqrt(max(rows, cols)).

    The arguments are those of ``torch.optim.Muon``; the arithmetic differs in that
    u is divided by |u|_F + eps (there max(|u|_F, eps)) and that the products
    take fp16 operands (there bf16). Parameters of more than two dimensions are
    stacks of matrices here: give a convolution's weight as a
    [out, in * height * width] view. ``ns_coefficients`` are limited as
    :func:`turboadam_b200.orthogonalize` says.

    Parameters: float32, bfloat16 or float16, at least two dimensions; the
    last two are the matrix. The momentum is kept in ``momentum_dtype``
    (float32 by default; bfloat16 halves it). u is rounded once to fp16
    (11 bits) before the products; the update is applied to the parameter
    from their fp32 sums.

    A step enqueues kernels only: it can be captured into a CUDA graph once
    the momentum exists and while the gradients keep their storage (the
    hyperparameters are captured by value). ``momentum_dtype`` is keyword-only
    and not part of ``torch.optim.Muon``.
    """

    def __init__(self, params, lr: float = 1e-3, weight_decay: float = 0.1,
                 momentum: float = 0.95, nesterov: bool = True,
                 ns_coefficients=NS_COEFFICIENTS, eps: float = NS_EPS, ns_steps: int = NS_STEPS,
                 adjust_lr_fn: str | None = None, *,
                 momentum_dtype: torch.dtype = torch.float32):
        if momentum_dtype not in (torch.float32, torch.bfloat16):
            raise ValueError("momentum_dtype must be float32 or bfloat16, got "
                             f"{momentum_dtype}")
        self._momentum_dtype = momentum_dtype
        defaults = dict(lr=lr, weight_decay=weight_decay, momentum=momentum, nesterov=nesterov,
                        ns_coefficients=ns_coefficients, eps=eps, ns_steps=ns_steps,
                        adjust_lr_fn=adjust_lr_fn)
        _check_group(defaults)
        super().__init__(params, defaults)

    def __getstate__(self):
        return {**super().__getstate__(), "_momentum_dtype": self._momentum_dtype}

    def add_param_group(self, param_group):
        super().add_param_group(param_group)
        try:
            _check_group(self.param_groups[-1])
            for p in self.param_groups[-1]["params"]:
                if p.dim() < 2:
                    raise ValueError("Muon updates matrices; a parameter has "
                                     f"{p.dim()} dimension(s): give it to TurboAdam")
        except Exception:
            self.param_groups.pop()
            raise

    def load_state_dict(self, state_dict):
        """torch casts state to the parameters' dtype; the momentum keeps its own."""
        saved = [s.get("momentum_buffer") if isinstance(s, dict) else None
                 for s in state_dict["state"].values()]
        index = dict(zip(state_dict["state"].keys(), saved))
        flat = [p for g in self.param_groups for p in g["params"]]
        ids = [i for g in state_dict["param_groups"] for i in g["params"]]
        for i, p in zip(ids, flat):
            m = index.get(i)
            if m is not None and m.shape != p.shape:
                raise ValueError(f"momentum of shape {tuple(m.shape)} for a parameter of shape "
                                 f"{tuple(p.shape)}")
        super().load_state_dict(state_dict)
        for i, p in zip(ids, flat):
            m = index.get(i)
            if m is not None:
                self.state[p]["momentum_buffer"] = (
                    m.detach().to(device=p.device, dtype=self._momentum_dtype, copy=True)
                    .contiguous())

    @torch.no_grad()
    def step(self, closure=None):
        """Perform a single optimization step."""
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group in self.param_groups:
            by_dev = {}
            for p in group["params"]:
                if p.grad is not None and p.numel():
                    _lib.require_cuda(p)
                    if p.dtype not in _DTYPES:
                        raise NotImplementedError(f"param dtype {p.dtype}: Muon is built for "
                                                  "float32, bfloat16 and float16")
                    if p.grad.is_sparse:
                        raise NotImplementedError("Muon does not take sparse gradients")
                    by_dev.setdefault(p.device, []).append(p)
            for dev, params in by_dev.items():
                self._step_device(group, dev, params)
        return loss

    def _fitting(self, p, dev):
        """The gradient and momentum of a parameter, as the kernels can take them: they read and
        write all three through pointers, at the parameter's size."""
        m, g = self.state[p].get("momentum_buffer"), p.grad
        if g.shape != p.shape or g.device != dev:
            raise ValueError(f"gradient {tuple(g.shape)} on {g.device} for a parameter "
                             f"{tuple(p.shape)} on {dev}")
        if g.dtype not in _DTYPES:
            raise NotImplementedError(f"grad dtype {g.dtype}")
        if m is None:
            m = torch.zeros(p.shape, dtype=self._momentum_dtype, device=dev)
        elif not isinstance(m, torch.Tensor):
            raise TypeError(f"momentum_buffer is a {type(m).__name__}, not a tensor")
        elif m.shape != p.shape or m.device != dev:
            raise ValueError(f"momentum {tuple(m.shape)} on {m.device} for a parameter "
                             f"{tuple(p.shape)} on {dev}")
        elif m.dtype not in _DTYPES:
            raise NotImplementedError(f"momentum dtype {m.dtype}")
        if not p.is_contiguous() or not m.is_contiguous():
            raise NotImplementedError("Muon updates contiguous parameters and momentum")
        self.state[p]["momentum_buffer"] = m
        return g, m

    def _step_device(self, group, dev, params):
        _check_adjustment(group["adjust_lr_fn"])
        options, coeffs = ortho_options(group["ns_coefficients"], group["ns_steps"], group["eps"],
                                        group["momentum"], group["nesterov"])
        lr = float(group["lr"])
        keep = 1.0 - lr * group["weight_decay"]
        alive, part, used = [], [], 0

        def flush():
            nonlocal part, used
            if part:
                run_ortho((_lib.TaOrthoTensor * len(part))(*part), len(part), options, dev)
            part, used = [], 0

        # all are checked before the first is changed
        fitting = [self._fitting(p, dev) for p in params]
        for p, (g, m) in zip(params, fitting):
            if not g.is_contiguous():
                g = g.contiguous()
            alive.append(g)
            rows, cols = p.shape[-2:]
            t = _lib.TaOrthoTensor()
            t.in_dev, t.momentum_dev, t.out_dev = g.data_ptr(), m.data_ptr(), p.data_ptr()
            t.batch, t.rows, t.cols = p.numel() // (rows * cols), rows, cols
            t.in_dtype, t.momentum_dtype = _DTYPES[g.dtype], _DTYPES[m.dtype]
            t.out_dtype, t.flags = _DTYPES[p.dtype], _lib.TA_ORTHO_UPDATE
            t.keep, t.gain = keep, _gain(group["adjust_lr_fn"], lr, rows, cols)
            # two scaled copies and three square matrices, 16-bit
            small = min(rows, cols)
            need = t.batch * (4 * rows * (cols + 8) + 6 * small * (small + 8))
            if part and used + need > WORKSPACE_LIMIT:
                flush()
            part.append(t)
            used += need
        flush()
        # written through pointers: graphs that saved them before the step notice
        torch.autograd.graph.increment_version(params)
        torch.autograd.graph.increment_version([m for _, m in fitting])
