"""Fused optimizer steps after backward for TimeMix's float32 parameters on MI355X: AdamW, and
orthogonalised updates for its matrices.

The reference updates each student layer after its backward with three torch steps
(train.py:202-208, optimizer from theseus/stage.py:39-42):

    for p in params: p.grad.mul_(world / count)
    norm = clip_grad_norm_(params, clip_norm, error_if_nonfinite=True)
    optimizer.step()        # torch.optim.AdamW(fused=True), groups decay / no decay

``FusedAdamW.step_after_backward(grad_scale, max_norm)`` does the same in one call of
``theseus_adamw_step`` (include/theseus_optim.h): per-chunk float64 sums of squared
gradients, a fixed-order final sum that forms the norm, the clip factor and a
non-finite flag in device memory, and the AdamW update reading that factor -- no
host synchronisation before the update, no scaled or clipped gradient written back,
deterministic results.  ``step()`` is plain AdamW (no scale, no clip), so the class is
also a drop-in ``torch.optim.AdamW`` for float32 CUDA parameters; its state uses
AdamW's keys ("step", "exp_avg", "exp_avg_sq"), so optimizer checkpoints keep their
format (theseus/checkpoint.py saves ``optimizer.state_dict()``), and LR schedulers
work on ``param_groups`` as usual.

``FusedMuon`` steps matrices along the orthogonal factor of their momentum (Muon) instead, with
the same two ways to call it, and ``orthogonalize`` is that factor alone (C ABI:
include/theseus_muon.h).  The reference trains with AdamW only.
"""
from __future__ import annotations

import ctypes
import functools
import math

import torch

from .fused import _direct
from .wkv7 import extension


class _Tensor(ctypes.Structure):  # theseus_adamw_tensor
    _fields_ = [("param", ctypes.c_void_p), ("grad", ctypes.c_void_p), ("exp_avg", ctypes.c_void_p),
                ("exp_avg_sq", ctypes.c_void_p), ("numel", ctypes.c_longlong), ("lr", ctypes.c_float),
                ("weight_decay", ctypes.c_float), ("step_size", ctypes.c_float),
                ("bias_correction2_sqrt", ctypes.c_float)]


class _Schulz(ctypes.Structure):  # theseus_newton_schulz
    _fields_ = [("steps", ctypes.c_int)] + [(n, ctypes.c_float) for n in ("a", "b", "c", "eps")]


class _Orth(ctypes.Structure):  # theseus_orthogonalize_matrix
    _fields_ = [("x", ctypes.c_void_p), ("out", ctypes.c_void_p), ("row_stride", ctypes.c_longlong), ("rows", ctypes.c_int),
                ("cols", ctypes.c_int), ("dtype", ctypes.c_int)]


class _Matrix(ctypes.Structure):  # theseus_muon_matrix
    _fields_ = [("param", ctypes.c_void_p), ("grad", ctypes.c_void_p), ("momentum", ctypes.c_void_p), ("rows", ctypes.c_int),
                ("cols", ctypes.c_int), ("keep", ctypes.c_float), ("step", ctypes.c_float)]


_bound = None


def _lib():
    global _bound
    lib = extension().lib
    if _bound is None:
        lib.theseus_adamw_workspace_size.argtypes = [ctypes.POINTER(_Tensor), ctypes.c_int]
        lib.theseus_adamw_workspace_size.restype = ctypes.c_size_t
        lib.theseus_adamw_step.argtypes = ([ctypes.POINTER(_Tensor), ctypes.c_int] + [ctypes.c_float] * 5
                                           + [ctypes.c_int, ctypes.c_void_p, ctypes.c_void_p, ctypes.c_size_t,
                                              ctypes.c_void_p])
        lib.theseus_adamw_step.restype = ctypes.c_int
        f32, i32, vp, sz = ctypes.c_float, ctypes.c_int, ctypes.c_void_p, ctypes.c_size_t
        lib.theseus_orthogonalize_workspace_size.argtypes = [ctypes.POINTER(_Orth), i32]
        lib.theseus_orthogonalize_workspace_size.restype = sz
        lib.theseus_orthogonalize.argtypes = [ctypes.POINTER(_Orth), i32, ctypes.POINTER(_Schulz), vp, sz, vp]
        lib.theseus_orthogonalize.restype = i32
        lib.theseus_muon_workspace_size.argtypes = [ctypes.POINTER(_Matrix), i32]
        lib.theseus_muon_workspace_size.restype = sz
        lib.theseus_muon_step.argtypes = [ctypes.POINTER(_Matrix), i32, ctypes.POINTER(_Schulz), ctypes.c_double, i32, f32, f32, i32, vp, vp, sz, vp]
        lib.theseus_muon_step.restype = i32
        _bound = True
    return lib


NONFINITE_MSG = ("The total norm of order 2.0 for gradients from `parameters` is non-finite, so it cannot be "
                 "clipped. To disable this error and scale the gradients by the non-finite norm anyway, set "
                 "`error_if_nonfinite=False`")


class FusedAdamW(torch.optim.Optimizer):
    """AdamW over float32 CUDA parameters with the reference's post-backward step fused in."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2):
        if not 0.0 <= lr:
            raise ValueError(f"Invalid learning rate: {lr}")
        if not 0.0 <= eps:
            raise ValueError(f"Invalid epsilon value: {eps}")
        if not 0.0 <= betas[0] < 1.0 or not 0.0 <= betas[1] < 1.0:
            raise ValueError(f"Invalid beta parameters: {betas}")
        if not 0.0 <= weight_decay:
            raise ValueError(f"Invalid weight_decay value: {weight_decay}")
        super().__init__(params, dict(lr=lr, betas=tuple(betas), eps=eps, weight_decay=weight_decay))

    # -- the tensor list ------------------------------------------------------------------
    def _entries(self):
        hyper, entries, keep, device = None, [], [], None
        for group in self.param_groups:
            h = (float(group["betas"][0]), float(group["betas"][1]), float(group["eps"]))
            if hyper is None:
                hyper = h
            elif h != hyper:
                raise ValueError("FusedAdamW: all parameter groups must share betas and eps")
            for p in group["params"]:
                if p.grad is None:
                    continue
                g = p.grad
                if not (p.is_cuda and p.dtype == torch.float32 and p.is_contiguous()):
                    raise RuntimeError("FusedAdamW: parameters must be contiguous float32 CUDA tensors")
                if g.is_sparse or not (g.dtype == torch.float32 and g.is_contiguous() and g.shape == p.shape
                                       and g.device == p.device):
                    raise RuntimeError("FusedAdamW: gradients must be dense contiguous float32 like the parameter")
                if device is None:
                    device = p.device
                elif p.device != device:
                    raise RuntimeError("FusedAdamW: all parameters must be on one device")
                st = self.state[p]
                if not st:
                    st["step"] = torch.tensor(0.0)
                    st["exp_avg"] = torch.zeros_like(p, memory_format=torch.preserve_format)
                    st["exp_avg_sq"] = torch.zeros_like(p, memory_format=torch.preserve_format)
                elif st["step"].device.type != "cpu":  # e.g. loaded from torch's fused AdamW
                    st["step"] = st["step"].detach().float().cpu()
                step = float(st["step"]) + 1.0
                lr, wd = float(group["lr"]), float(group["weight_decay"])
                bc1 = 1.0 - hyper[0] ** step
                bc2 = 1.0 - hyper[1] ** step
                entries.append(_Tensor(p.data_ptr(), g.data_ptr(), st["exp_avg"].data_ptr(),
                                       st["exp_avg_sq"].data_ptr(), p.numel(), lr, wd, lr / bc1, math.sqrt(bc2)))
                keep.append(st)
        return hyper, entries, keep, device

    def _run(self, grad_scale, max_norm, error_if_nonfinite):
        hyper, entries, states, device = self._entries()
        if not entries:
            return None
        lib = _lib()
        arr = (_Tensor * len(entries))(*entries)
        norm_mode = max_norm is not None
        ws_bytes = int(lib.theseus_adamw_workspace_size(arr, len(entries))) if norm_mode else 0
        ws = torch.empty(max(ws_bytes, 8), dtype=torch.uint8, device=device)
        result = torch.empty(3, dtype=torch.float32, device=device)
        with torch.cuda.device(device):
            status = lib.theseus_adamw_step(
                arr, len(entries), float(grad_scale), float(max_norm) if norm_mode else -1.0,
                hyper[0], hyper[1], hyper[2], 1 if error_if_nonfinite else 0,
                ctypes.c_void_p(result.data_ptr()), ctypes.c_void_p(ws.data_ptr()), ctypes.c_size_t(ws_bytes),
                ctypes.c_void_p(torch.cuda.current_stream(device).cuda_stream))
        if status:
            raise RuntimeError("theseus_adamw: " + lib.theseus_wkv7_error_string(status).decode())
        if norm_mode and error_if_nonfinite and bool(result[2].item()):
            raise RuntimeError(NONFINITE_MSG)  # (the kernels left every parameter unchanged)
        for st in states:
            st["step"] += 1.0
        return result[0] if norm_mode else None

    # -- public ----------------------------------------------------------------------------
    @torch.no_grad()
    def step(self, closure=None):
        """torch.optim.AdamW's step for every parameter with a gradient."""
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        self._run(1.0, None, False)
        return loss

    @torch.no_grad()
    def step_after_backward(self, grad_scale=1.0, max_norm=None, error_if_nonfinite=True):
        """The reference's ``p.grad.mul_(grad_scale)`` loop, ``clip_grad_norm_(params,
        max_norm, error_if_nonfinite)`` and ``step()`` in one fused call
        (train.py:202-208).  Returns the total norm of the scaled gradients as a 0-d
        CUDA tensor, like clip_grad_norm_ (None when ``max_norm`` is None: no clipping
        and no norm).  The gradients themselves are left as they were.  With
        ``error_if_nonfinite`` a non-finite norm raises clip_grad_norm_'s RuntimeError
        and no parameter, moment or step count changes (this reads one flag back, a
        synchronisation the reference makes too); otherwise the update runs with the
        non-finite factor, as in torch."""
        return self._run(grad_scale, max_norm, error_if_nonfinite)


# ------------------------------------------------------------------------------ orthogonalised updates
COEFFICIENTS = (3.4445, -4.7750, 2.0315)  # of the usual five steps: singular values to 0.68 .. 1.21 in few of them
_MAX_SIDE, _MAX_STRIDE = 1 << 17, 1 << 21  # include/theseus_muon.h


@functools.lru_cache(maxsize=64)
def _in_range(steps, a, b, c):
    """Whether singular values from 0 .. 1 stay in what float16 products hold: the largest in 1/4 .. 3 until the last step,
    |a + b s^2 + c s^4| up to 32 (a grid of 512, so 1 % of room)."""
    largest = 1.0
    for _ in range(steps):
        if not .25 <= largest <= 2.97:
            return False
        grid = [largest * i / 512 for i in range(513)]
        factors = [abs(a + (b + c * s * s) * s * s) for s in grid]
        if max(factors) > 31.7:
            return False
        largest = max(s * f for s, f in zip(grid, factors))
    return True


def _schulz(steps, coefficients, eps):
    if not 1 <= steps <= 100:
        raise ValueError(f"theseus_muon: steps must be in 1 .. 100, got {steps}")
    if len(coefficients) != 3 or not all(math.isfinite(c) and abs(c) < 1e6 for c in coefficients):
        raise ValueError(f"theseus_muon: expected three finite coefficients, got {coefficients}")
    if not 0 <= eps <= 3.4028234663852886e38:
        raise ValueError(f"theseus_muon: eps must not be negative, and finite in float32, got {eps}")
    if not _in_range(int(steps), *(float(c) for c in coefficients)):
        raise ValueError(f"theseus_muon: {steps} steps with coefficients {coefficients} leave float16's range (largest singular values "
                         "out of 1/4 .. 3, or factors above 32)")
    return _Schulz(int(steps), *(float(c) for c in coefficients), float(eps))


def _run_muon(device, work, call):
    """``call(workspace, bytes, stream)`` of a status, on the device with ``work`` bytes."""
    ws = torch.empty(max(work, 8), dtype=torch.uint8, device=device)
    with torch.cuda.device(device):
        status = call(ws.data_ptr(), work, torch.cuda.current_stream(device).cuda_stream)
    if status:
        raise RuntimeError("theseus_muon: " + extension().lib.theseus_wkv7_error_string(status).decode())


@torch.no_grad()
def orthogonalize(x, *, steps=5, coefficients=COEFFICIENTS, eps=1e-7):
    """The matrices' singular values brought near 1, their singular vectors kept (Newton-Schulz):

        X = x / max(|x|_F, eps);  steps times: A = X X^T, X = a X + (b A + c A^2) X

    (on the short side; the norm per matrix).  x: a tensor [..., m, n] (leading dimensions: that many
    matrices) or a list of them, bfloat16 or float32, sides up to 2^17; rows may lie apart.  Returns
    bfloat16 tensors of the same shapes (a list for a list).  With the usual coefficients and steps, singular values from
    1.5e-3 of the norm on end anywhere in 0.68 .. 1.21, smaller ones are raised by up to 485; other coefficients are taken that
    keep the largest ones in 1/4 .. 3 and |a + b s^2 + c s^4| below 32.  Norms below 1e-30 count as 1e-30 where eps is less.  All
    matrices share the launches.  The products take float16 operands and add in float32, X is held in 22 bits: in the usual steps
    off by 2e-3 to 3e-3 of the exact polynomial's norm, 1.7e-3 of it the result's rounding (more steps of these coefficients do not
    converge and add to it: 3e-3 after ten, 5e-3 after twenty).  The same list gives the same bits on every run (in another
    list a matrix' sums may be cut otherwise).  A matrix with a value that is not finite comes back NaN.  Not differentiable;
    not for traces, functorch transforms or forward mode."""
    ns = _schulz(steps, coefficients, eps)
    xs = [x] if isinstance(x, torch.Tensor) else list(x)
    if not xs:
        return []
    if not _direct(*xs):
        raise RuntimeError("theseus_muon: orthogonalize has no forward-mode derivative, and no trace or functorch transform takes it in")
    outs, entries, held, device = [], [], [], xs[0].device
    for t in xs:
        if not t.is_cuda:
            raise ValueError("theseus_muon: matrices must be CUDA tensors")
        if t.device != device:
            raise ValueError(f"theseus_muon: all matrices must be on {device}, got {t.device}")
        if t.dtype not in (torch.bfloat16, torch.float32):
            raise TypeError(f"theseus_muon: matrices must be bfloat16 or float32, got {t.dtype}")
        if t.dim() < 2 or max(t.shape[-2:]) > _MAX_SIDE:
            raise ValueError(f"theseus_muon: expected [..., m, n] with sides up to 2^17, got {list(t.shape)}")
        out = torch.empty(t.shape, dtype=torch.bfloat16, device=device)
        outs.append(out)
        if not t.numel():
            continue
        m, n = t.shape[-2:]
        t = t.detach().reshape(-1, m, n)
        if t.stride(2) != 1 and n > 1 or m > 1 and not n <= t.stride(1) <= _MAX_STRIDE:
            t = t.contiguous()
        held.append(t)  # (until the call has been made)
        apart, size, at, to = t.stride(0) * t.element_size(), 2 * m * n, t.data_ptr(), out.data_ptr()
        dtype, row = int(t.dtype == torch.float32), max(t.stride(1), n)
        entries += [_Orth(at + i * apart, to + i * size, row, m, n, dtype) for i in range(t.shape[0])]
    if entries:
        lib, count = _lib(), len(entries)
        arr = (_Orth * count)(*entries)
        _run_muon(device, int(lib.theseus_orthogonalize_workspace_size(arr, count)),
                  lambda ws, nbytes, stream: lib.theseus_orthogonalize(arr, count, ctypes.byref(ns), ws, nbytes, stream))
    return outs[0] if isinstance(x, torch.Tensor) else outs


class FusedMuon(torch.optim.Optimizer):
    """Momentum, its orthogonalised direction, weight decay and step over float32 CUDA matrices:

        momentum_buffer = mu momentum_buffer + (1 - mu) g
        u = mu momentum_buffer + (1 - mu) g          (without nesterov: momentum_buffer)
        p = p (1 - lr weight_decay) - lr size(p) orthogonalize(u)

    size(p) of a [m, n] matrix is sqrt(max(1, m / n)) with scale="shape" and 0.2 sqrt(max(m, n)) with
    scale="rms", updates of about the size of AdamW's.  For the matrices inside the layers;
    embeddings, heads and vectors are FusedAdamW's.  The orthogonalised direction is not rounded to bfloat16
    here: it goes from the last product's float32 sums into the parameter.  State key "momentum_buffer"."""

    def __init__(self, params, lr=1e-3, weight_decay=0.1, momentum=0.95, nesterov=True, coefficients=COEFFICIENTS, eps=1e-7, steps=5,
                 scale="shape"):
        if not 0.0 <= lr:
            raise ValueError(f"Invalid learning rate: {lr}")
        if not 0.0 <= weight_decay:
            raise ValueError(f"Invalid weight_decay value: {weight_decay}")
        if not 0.0 <= momentum < 1.0:
            raise ValueError(f"Invalid momentum value: {momentum}")
        _schulz(steps, coefficients, eps)
        super().__init__(params, dict(lr=lr, weight_decay=weight_decay, momentum=momentum, nesterov=nesterov,
                                      coefficients=tuple(coefficients), eps=eps, steps=steps, scale=scale))

    def add_param_group(self, group):
        super().add_param_group(group)
        group = self.param_groups[-1]
        if group["scale"] not in ("shape", "rms"):
            raise ValueError(f"FusedMuon: unknown scale {group['scale']!r} (shape or rms)")
        for p in group["params"]:
            if p.dim() != 2 or max(p.shape) > _MAX_SIDE:
                raise ValueError(f"FusedMuon: parameters must be matrices with sides up to 2^17, got {list(p.shape)}")

    def _entries(self):
        hyper, entries, device = None, [], None
        for group in self.param_groups:
            h = (float(group["momentum"]), bool(group["nesterov"]), tuple(group["coefficients"]), float(group["eps"]), int(group["steps"]))
            if hyper is None:
                hyper = h
            elif h != hyper:
                raise ValueError("FusedMuon: all parameter groups must share momentum, nesterov, coefficients, eps and steps")
            lr, keep = float(group["lr"]), 1.0 - float(group["lr"]) * float(group["weight_decay"])
            rms = group["scale"] == "rms"
            for p in group["params"]:
                g = p.grad
                if g is None:
                    continue
                if not (p.is_cuda and p.dtype == torch.float32 and p.is_contiguous()):
                    raise RuntimeError("FusedMuon: parameters must be contiguous float32 CUDA tensors")
                if g.is_sparse or not (g.dtype == torch.float32 and g.is_contiguous() and g.shape == p.shape and g.device == p.device):
                    raise RuntimeError("FusedMuon: gradients must be dense contiguous float32 like the parameter")
                if device is None:
                    device = p.device
                elif p.device != device:
                    raise RuntimeError("FusedMuon: all parameters must be on one device")
                state = self.state[p]
                if not state:
                    state["momentum_buffer"] = torch.zeros_like(p, memory_format=torch.preserve_format)
                buf = state["momentum_buffer"]
                if not (buf.dtype == torch.float32 and buf.is_contiguous() and buf.shape == p.shape and buf.device == p.device):
                    raise RuntimeError("FusedMuon: momentum_buffer must be contiguous float32 like the parameter")
                m, n = p.shape
                if not m or not n:
                    continue
                size = .2 * math.sqrt(max(m, n)) if rms else math.sqrt(max(1.0, m / n))
                entries.append(_Matrix(p.data_ptr(), g.data_ptr(), buf.data_ptr(), m, n, keep, lr * size))
        return hyper, entries, device

    def _run(self, grad_scale, max_norm, error_if_nonfinite):
        hyper, entries, device = self._entries()
        norm, limit = max_norm is not None, -1.0 if max_norm is None else float(max_norm)
        if device is None or not (entries or norm):
            return None
        if not entries and not limit >= 0:  # (nothing to step, and no norm)
            return torch.full((), math.nan, device=device)
        momentum, nesterov, coefficients, eps, steps = hyper
        ns, lib, count = _schulz(steps, coefficients, eps), _lib(), len(entries)
        arr = (_Matrix * count)(*entries)
        result = torch.empty(3, dtype=torch.float32, device=device) if norm else None
        _run_muon(device, int(lib.theseus_muon_workspace_size(arr, count)),
                  lambda ws, nbytes, stream: lib.theseus_muon_step(
                      arr, count, ctypes.byref(ns), momentum, int(nesterov), float(grad_scale), limit,
                      int(error_if_nonfinite), result.data_ptr() if norm else None, ws, nbytes, stream))
        if norm and error_if_nonfinite and bool(result[2].item()):
            raise RuntimeError(NONFINITE_MSG)  # (the kernels left every parameter unchanged)
        return result[0] if norm else None

    @torch.no_grad()
    def step(self, closure=None):
        """A step for every parameter with a gradient."""
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        self._run(1.0, None, False)
        return loss

    @torch.no_grad()
    def step_after_backward(self, grad_scale=1.0, max_norm=None, error_if_nonfinite=True):
        """``step`` on the gradients times ``grad_scale``, clipped to ``max_norm`` over this optimizer's
        parameters: FusedAdamW.step_after_backward's arguments, result and errors.  (Scaling all of a run's
        gradients alike changes nothing but eps' part; clipping weighs this step's against the momentum.  A step that
        is left out for its norm may take as long as any other.)"""
        return self._run(grad_scale, max_norm, error_if_nonfinite)
