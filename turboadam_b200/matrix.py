"""Matrix operators beside the packed optimizer step (include/turboadam_b200_matrix.h).

* :func:`linear_act` -- a linear layer with bias, activation and residual in
  its product's epilogue, and its gradients;
* :func:`orthogonalize` -- the Newton-Schulz iteration of the Muon optimizer;
* :class:`turboadam_b200.Muon` (muon.py) -- the optimizer step built on it.

Like the optimizer, they run on CUDA (sm_100a) tensors only; there is no CPU
fallback. None has a counterpart in the reference.
"""
from __future__ import annotations

import ctypes
import math
import struct
import threading

import torch
from torch.autograd import forward_ad

from . import _lib

# the quintic of the Muon optimizer, tuned for slope at zero
NS_COEFFICIENTS = (3.4445, -4.7750, 2.0315)
NS_STEPS = 5
NS_EPS = 1e-7

_DTYPES = {torch.float32: _lib.TA_F32, torch.bfloat16: _lib.TA_BF16, torch.float16: _lib.TA_F16}
_HALF = (torch.bfloat16, torch.float16)
_ACTIVATIONS = {None: _lib.TA_ACT_NONE, "none": _lib.TA_ACT_NONE, "relu": _lib.TA_ACT_RELU,
                "gelu": _lib.TA_ACT_GELU, "gelu_tanh": _lib.TA_ACT_GELU_TANH,
                "silu": _lib.TA_ACT_SILU}

# device index -> status word that every call on that device ORs into, and the tensor that holds it.
# It lies in pinned host memory, which kernels reach at the same address: they write it only when a
# wait has run out, and a call sees what earlier ones have left there without synchronising.
_words = {}
_words_lock = threading.Lock()


def _word(index: int) -> int:
    """Address of the device's status word. Raises if an earlier call's results are void."""
    at = _words.get(index)
    if at is None:
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("the first call on a device must run outside CUDA graph capture")
        with _words_lock:
            if index not in _words:
                st = torch.zeros(1, dtype=torch.int32, pin_memory=True)
                _words[index] = ctypes.c_uint32.from_address(st.data_ptr()), st
            at = _words[index]
    if at[0].value:
        raise _lib.TurboAdamBackendError(
            f"a bounded wait of an earlier call on cuda:{index} ran out (status "
            f"{at[0].value:#x}): its results are void. matrix.read_status() clears this")
    return at[1].data_ptr()


def read_status(clear: bool = True) -> int:
    """Device status bits of the matrix operators since the last read, over
    all devices (TA_STATUS_WAIT_TIMEOUT: a bounded wait ran out and that
    call's results are void; calls raise until the bit has been cleared).
    Synchronises."""
    out = 0
    for idx, (word, _) in list(_words.items()):
        torch.cuda.synchronize(idx)
        out |= word.value
        if clear:
            word.value = 0
    return out


def check_coefficients(coefficients, steps: int):
    """One (a, b, c), or one per step, as a flat list of 3 * steps floats."""
    if isinstance(steps, bool) or int(steps) != steps or not 1 <= steps <= 32:
        raise ValueError(f"steps must be a whole number from 1 to 32, got {steps}")
    rows = list(coefficients)
    if len(rows) == 3 and not any(hasattr(r, "__len__") for r in rows):
        rows = [rows] * int(steps)
    if len(rows) != steps or any(not hasattr(r, "__len__") or len(r) != 3 for r in rows):
        raise ValueError("coefficients must be one (a, b, c) or one (a, b, c) per step")
    return [float(v) for r in rows for v in r]


def ortho_options(coefficients, steps, eps, momentum=0.0, nesterov=False):
    """The ABI options, and the host array they point at."""
    if not eps >= 0:
        raise ValueError(f"eps must not be negative, got {eps}")
    flat = check_coefficients(coefficients, steps)
    arr = (ctypes.c_double * len(flat))(*flat)
    return _lib.TaOrthoOptions(ctypes.cast(arr, ctypes.c_void_p), int(steps), int(nesterov),
                               float(eps), float(momentum)), arr


def _no_tangents(what, *tensors):
    """The operators read data pointers, past a forward-mode tangent."""
    for t in tensors:
        if t is not None and forward_ad.unpack_dual(t).tangent is not None:
            raise NotImplementedError(f"{what}: forward-mode derivatives are not built")


class _On:
    """``with _On(index):`` the calls inside see that device as the current one."""

    __slots__ = ("index", "before")

    def __init__(self, index):
        self.index = index

    def __enter__(self):
        self.before = torch._C._cuda_getDevice()
        if self.before != self.index:
            torch._C._cuda_setDevice(self.index)

    def __exit__(self, *exc):
        if self.before != self.index:
            torch._C._cuda_setDevice(self.before)


def _call(size_fn, fn, what, args, dev):
    """One call of the library on the current stream of ``dev``: its workspace, sized by
    ``size_fn``, is allocated on that stream, so it is reused only for work ordered after the
    call."""
    index = dev.index
    with _On(index):
        need = size_fn(*args)
        if need == 0:
            why = _lib.load().ta_last_error()
            if why:
                raise _lib.TurboAdamBackendError(
                    f"{what} failed: {why.decode(errors='replace')}")
        word = _word(index)
        ws = torch.empty(need, dtype=torch.uint8, device=dev)
        rc = fn(*args, ws.data_ptr(), need, word, torch._C._cuda_getCurrentRawStream(index))
    if rc:
        _lib.check(rc, what)


def run_ortho(table, n, options, dev):
    """One ta_orthogonalize call on the current stream of ``dev``."""
    lib = _lib.load()
    _call(lib.ta_ortho_workspace_size, lib.ta_orthogonalize, "ta_orthogonalize",
          (table, n, ctypes.byref(options)), dev)


@torch.no_grad()
def orthogonalize(x: torch.Tensor, steps: int = NS_STEPS, coefficients=NS_COEFFICIENTS,
                  eps: float = NS_EPS, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """Newton-Schulz orthogonalisation of a matrix or a stack of matrices.

    With X = x / (|x|_F + eps) and, ``steps`` times, A = X X^T (X^T X for a
    tall matrix), X <- (a I + b A + c A^2) X; returns X in ``dtype``.
    ``coefficients`` is one (a, b, c), by default the Muon quintic, or one per
    step. x: float32, bfloat16 or float16, [..., rows, cols].

    The products take fp16 operands and fp32 sums. A 16-bit x enters
    unrounded, a 32-bit one as a pair of fp16 numbers (of which the first A
    sees the upper one). The result is off from the exact iteration by 0.8e-3
    to 2e-3 in the Frobenius norm and 1.5e-3 to 5e-3 in the 2-norm (gradients
    and random matrices with 70 to 14336 rows), so float32 outputs carry about
    nine good bits; fewer where a matrix of a few rows is close to singular
    (random 2 x 2: 1.6e-3 at the median, 1.7e-2 for one in a hundred). A zero matrix gives
    zero; a matrix with a NaN or an infinity gives NaN throughout.

    ``coefficients`` have to keep singular values below 8, and each step's
    polynomial and the product of two that act as a pair (the first two
    steps'; all pairs' where the shorter side is 2048 or more) below 255, or
    fp16 overflows and the result is NaN. The quintic stays under 1.3 and 12.

    Not differentiable: the result is detached from an x that requires a
    gradient, and an x with a forward-mode tangent is refused.
    """
    _lib.require_cuda(x)
    if forward_ad._current_level >= 0:
        _no_tangents("orthogonalize", x)
    if x.dim() < 2:
        raise ValueError(f"orthogonalize takes matrices, got {x.dim()} dimension(s)")
    if x.dtype not in _DTYPES or dtype not in _DTYPES:
        raise NotImplementedError(f"orthogonalize: dtypes {x.dtype} -> {dtype} (float32, bfloat16 "
                                  "and float16 are built)")
    options, keep = ortho_options(coefficients, steps, eps)
    src = x.contiguous()
    out = torch.empty(x.shape, dtype=dtype, device=x.device)
    if out.numel() == 0:
        return out
    rows, cols = x.shape[-2:]
    table = (_lib.TaOrthoTensor * 1)()
    t = table[0]
    t.in_dev, t.out_dev = src.data_ptr(), out.data_ptr()
    t.batch, t.rows, t.cols = x.numel() // (rows * cols), rows, cols
    t.in_dtype, t.out_dtype = _DTYPES[x.dtype], _DTYPES[dtype]
    t.flags = _lib.TA_ORTHO_PAIR
    run_ortho(table, 1, options, x.device)
    return out


def _two_strides(t: torch.Tensor) -> torch.Tensor:
    """A matrix the products can read: one unit stride, lines that do not overlap."""
    (r, c), (sr, sc) = t.shape, t.stride()
    if (c <= 1 or sc == 1) and (r <= 1 or sr >= c):
        return t
    if (r <= 1 or sr == 1) and (c <= 1 or sc >= r):
        return t
    return t.contiguous()


def _rows(t: torch.Tensor) -> torch.Tensor:
    """A matrix with unit column stride and rows that do not overlap."""
    (r, c), (sr, sc) = t.shape, t.stride()
    return t if (c <= 1 or sc == 1) and (r <= 1 or sr >= c) else t.contiguous()


# ta_linear and ta_linear_grad (include/turboadam_b200_matrix.h), packed in one go
_LINEAR = struct.Struct("@6P3q2q2q2q4i")
_LINEAR_GRAD = struct.Struct("@7P3qq2q2q2q2i")


def _forward(x, w, bias, act, residual, need_deriv):
    lib = _lib.load()
    x, w = _two_strides(x), _two_strides(w)
    (tokens, fan_in), fan_out = x.shape, w.shape[0]
    dev = x.device
    y = torch.empty((tokens, fan_out), dtype=x.dtype, device=dev)
    deriv = None
    if need_deriv:
        deriv = torch.empty((tokens, (fan_out + 7) // 8 * 8), dtype=torch.int16, device=dev)
    if tokens == 0 or fan_out == 0:
        return y, deriv
    if bias is not None:
        bias = bias.contiguous()
    if residual is not None:
        residual = _rows(residual)
    op = _LINEAR.pack(
        x.data_ptr(), w.data_ptr(), 0 if bias is None else bias.data_ptr(),
        0 if residual is None else residual.data_ptr(), y.data_ptr(),
        0 if deriv is None else deriv.data_ptr(), tokens, fan_in, fan_out, *x.stride(),
        *w.stride(), 0 if residual is None else residual.stride(0), fan_out, _DTYPES[x.dtype],
        0 if bias is None else _DTYPES[bias.dtype], act, 0)
    _call(lib.ta_linear_workspace_size, lib.ta_linear_forward, "ta_linear_forward", (op,), dev)
    return y, deriv


class _LinearAct(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, bias, residual, act):
        # the derivative is needed by every gradient but the residual's
        nx, nw, nb, _, _ = ctx.needs_input_grad
        need = act != _lib.TA_ACT_NONE and (nx or nw or nb)
        y, deriv = _forward(x, w, bias, act, residual, need)
        ctx.bias_dtype = None if bias is None else bias.dtype
        ctx.save_for_backward(x if nw else None, w if nx else None, deriv)
        ctx.dims = (*x.shape, w.shape[0])
        # the weight's gradient is laid out as the weight: input by output if its rows are
        ctx.io = w.stride(0) == 1 and w.stride(1) != 1
        return y

    @staticmethod
    def backward(ctx, dy):
        if torch.is_grad_enabled():  # create_graph=True
            raise NotImplementedError("linear_act is differentiable once")
        nx, nw, nb, nr, _ = ctx.needs_input_grad
        dx = dw = db = None
        if nx or nw or nb:
            lib = _lib.load()
            x, w, deriv = ctx.saved_tensors
            tokens, fan_in, fan_out = ctx.dims
            dev, dtype = dy.device, dy.dtype
            g = _rows(dy)
            xs = ws = dws = (0, 0)
            xp = wp = 0
            if nx:
                w = _two_strides(w)
                wp, ws = w.data_ptr(), w.stride()
                dx = torch.empty((tokens, fan_in), dtype=dtype, device=dev)
            if nw:
                x = _two_strides(x)
                xp, xs = x.data_ptr(), x.stride()
                if ctx.io:
                    dw = torch.empty((fan_in, fan_out), dtype=dtype, device=dev).t()
                else:
                    dw = torch.empty((fan_out, fan_in), dtype=dtype, device=dev)
                dws = dw.stride()
            if nb:
                db = torch.empty(fan_out, dtype=ctx.bias_dtype, device=dev)
            op = _LINEAR_GRAD.pack(
                g.data_ptr(), 0 if deriv is None else deriv.data_ptr(), xp, wp,
                0 if dx is None else dx.data_ptr(), 0 if dw is None else dw.data_ptr(),
                0 if db is None else db.data_ptr(), tokens, fan_in, fan_out,
                max(g.stride(0), fan_out), *xs, *ws, *dws, _DTYPES[dtype],
                0 if db is None else _DTYPES[db.dtype])
            _call(lib.ta_linear_backward_workspace_size, lib.ta_linear_backward,
                  "ta_linear_backward", (op,), dev)
        return dx, dw, db, dy if nr else None, None


def linear_act(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None,
               activation: str | None = None,
               residual: torch.Tensor | None = None) -> torch.Tensor:
    """``activation(x @ weight.T + bias) + residual`` as one product.

    x: [..., fan_in], weight: [fan_out, fan_in] (a transposed view of an
    input-by-output weight is read as it lies), bias: [fan_out], residual:
    [..., fan_out]; activation: None, "relu", "gelu", "gelu_tanh" or "silu".
    x, weight and residual are all bfloat16 or all float16; the bias may also
    be float32. Sums, bias, activation and residual are in fp32 and rounded
    once.

    Differentiable once in x, weight, bias and residual, in reverse mode. For the backward pass
    the activation's derivative is kept in 16 bits, to half of the operand
    type's rounding relative to itself; dz = dy * derivative is rounded once to
    the operand type for the two products that read it. A weight's gradient has the weight's layout.
    """
    if not x.is_cuda:
        _lib.require_cuda(x)
    act = _ACTIVATIONS.get(activation)
    if act is None:
        raise ValueError(f"activation must be one of {sorted(k for k in _ACTIVATIONS if k)} or "
                         f"None, got {activation!r}")
    if x.dtype not in _HALF:
        raise NotImplementedError(f"linear_act is built for bfloat16 and float16, got {x.dtype}")
    if x.dim() < 1 or weight.dim() != 2 or x.shape[-1] != weight.shape[1]:
        raise ValueError(f"x {tuple(x.shape)} and weight {tuple(weight.shape)} do not match: "
                         "[..., fan_in] and [fan_out, fan_in] are wanted")
    fan_in, fan_out = weight.shape[1], weight.shape[0]
    shape = (*x.shape[:-1], fan_out)
    dtype, device = x.dtype, x.device
    if weight.dtype != dtype or weight.device != device:
        raise ValueError(f"weight is {weight.dtype} on {weight.device}, x {dtype} on {device}")
    grad = x.requires_grad or weight.requires_grad
    if bias is not None:
        if bias.device != device or (bias.dtype != dtype and bias.dtype != torch.float32):
            raise ValueError(f"bias is {bias.dtype} on {bias.device}, x {dtype} on {device}")
        if bias.dim() != 1 or bias.shape[0] != fan_out:
            raise ValueError(f"bias has shape {tuple(bias.shape)}, wanted {(fan_out,)}")
        grad = grad or bias.requires_grad
    if residual is not None:
        if residual.dtype != dtype or residual.device != device:
            raise ValueError(f"residual is {residual.dtype} on {residual.device}, x {dtype} on "
                             f"{device}")
        if residual.shape != shape:
            raise ValueError(f"residual has shape {tuple(residual.shape)}, wanted {shape}")
        grad = grad or residual.requires_grad
    if forward_ad._current_level >= 0:
        _no_tangents("linear_act", x, weight, bias, residual)
    flat = x.dim() == 2
    if not flat:
        tokens = math.prod(x.shape[:-1])
        x = x.reshape(tokens, fan_in)
        if residual is not None:
            residual = residual.reshape(tokens, fan_out)
    if grad and torch.is_grad_enabled():
        y = _LinearAct.apply(x, weight, bias, residual, act)
    else:
        y, _ = _forward(x, weight, bias, act, residual, False)
    return y if flat else y.reshape(shape)
