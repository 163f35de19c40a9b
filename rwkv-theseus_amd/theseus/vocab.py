"""What a language model's head is trained on and answers with, over a large vocabulary
(C ABI: include/theseus_vocab.h).

The reference distils its student layers against hidden states and checks the converted model by
a divergence over full logits (theseus/losses.py:5-30, validate.py).  These operators are what
training the whole student takes next: losses on the head's output that never hold the
[tokens, vocabulary] logits, and the few logits of a teacher that are worth keeping.

* ``linear_cross_entropy(hidden, weight, labels)``: softmax cross entropy of hidden @ weight.T;
* ``linear_top_distillation(hidden, weight, top_values, top_indices)``: the divergence of the
  student's softmax from a teacher of whom each token's top logits are known;
* ``top_logits(logits, k)``: those top logits and indices, and the row's log-sum-exp.

The losses are differentiable in ``hidden`` and ``weight`` (bfloat16; under autocast other types
are cast as ``torch.nn.functional.linear`` casts them).  With ``reduction="mean"`` or ``"sum"``
the gradients are made together with the loss, in three products, and the backward multiplies
them by the upstream gradient; with ``"none"`` the backward makes them, from 16-bit exponentials
that the forward keeps where they take at most 256 MiB, and else from the logits formed again.
A second backward through the same loss (retain_graph) makes the gradients anew.  Where a backward
reads labels or a teacher's tensors again, it raises if they were changed in place since the call.
"""
from __future__ import annotations

import ctypes
import math

import torch

from .fused import _direct
from .wkv7 import _native, extension

MAX_TOP = 256  # THESEUS_VOCAB_MAX_TOP
MAX_STRIDE = 1 << 21  # elements from row to row of a weight (include/theseus_vocab.h)
_REDUCTIONS = {"none": 0, "sum": 1, "mean": 2}
_DTYPES = {torch.bfloat16: 0, torch.float32: 1}


class LossArgs(ctypes.Structure):
    """theseus_vocab_loss_args."""
    _fields_ = ([(n, ctypes.c_longlong) for n in ("rows", "vocab")] + [(n, ctypes.c_int) for n in ("width", "targets")]
                + [(n, ctypes.c_void_p) for n in ("hidden", "weight")]
                + [(n, ctypes.c_longlong) for n in ("hidden_stride", "weight_stride")]
                + [(n, ctypes.c_void_p) for n in ("index", "top_values")]
                + [(n, ctypes.c_int) for n in ("top_dtype", "reduction")]
                + [(n, ctypes.c_void_p) for n in ("teacher_lse", "row_weight")]
                + [("ignore_index", ctypes.c_longlong), ("temperature", ctypes.c_float)]
                + [(n, ctypes.c_void_p) for n in ("loss", "row_grad", "dhidden", "dweight")]
                + [("piece_rows", ctypes.c_longlong), ("kept", ctypes.c_void_p), ("phase", ctypes.c_int)])


_bound = None


def _lib():
    global _bound
    lib = extension().lib
    if _bound is None:
        vp, i32, i64, sz, f32 = ctypes.c_void_p, ctypes.c_int, ctypes.c_longlong, ctypes.c_size_t, ctypes.c_float
        lib.theseus_vocab_loss_workspace_size.argtypes = [ctypes.POINTER(LossArgs)]
        lib.theseus_vocab_loss_workspace_size.restype = sz
        lib.theseus_vocab_loss_kept_size.argtypes = [ctypes.POINTER(LossArgs)]
        lib.theseus_vocab_loss_kept_size.restype = sz
        lib.theseus_vocab_loss.argtypes = [ctypes.POINTER(LossArgs), vp, sz, vp]
        lib.theseus_vocab_loss.restype = i32
        lib.theseus_vocab_scale.argtypes = [vp, i64, vp, i64, vp, vp]
        lib.theseus_vocab_scale.restype = i32
        lib.theseus_vocab_top_workspace_size.argtypes = [i64, i64, i32, i32]
        lib.theseus_vocab_top_workspace_size.restype = sz
        lib.theseus_vocab_top.argtypes = [i64, i64, i32, i32, f32, vp, i64, vp, vp, vp, vp, sz, vp]
        lib.theseus_vocab_top.restype = i32
        _bound = True
    return lib


def _check(status):
    if status:
        raise RuntimeError("theseus_vocab: " + extension().lib.theseus_wkv7_error_string(status).decode())


def _stream(device):
    return torch.cuda.current_stream(device).cuda_stream


class _Call:
    """One loss's inputs, checked and laid out for theseus_vocab_loss."""

    def __init__(self, hidden, weight, index, top_values, teacher_lse, row_weight, ignore_index, temperature, reduction,
                 piece_rows):
        self.index, self.top_values, self.teacher_lse, self.row_weight = index, top_values, teacher_lse, row_weight
        self.ignore_index, self.temperature, self.reduction = ignore_index, temperature, reduction
        self.piece_rows, self.targets = piece_rows, 1 if top_values is None else top_values.shape[1]
        self.rows, self.vocab, self.width = hidden.shape[0], weight.shape[0], hidden.shape[1]
        self.device = hidden.device

    _HELD = {"index": "labels (or top_indices)", "top_values": "top_values", "teacher_lse": "teacher_lse", "row_weight": "token_weight"}

    def hold(self):
        """For a backward that forms the logits again: what it reads of the targets and that it was not changed
        since (unchanged).  Not saved_tensors, whose unpacking would ask that of every backward.  Tensors of
        inference mode have no version: a copy."""
        for name in self._HELD:
            t = getattr(self, name)
            if t is not None and t.is_inference():
                setattr(self, name, t.clone())
        self.versions = {name: getattr(self, name)._version for name in self._HELD if getattr(self, name) is not None}

    def unchanged(self):
        for name, version in self.versions.items():
            if getattr(self, name)._version != version:
                raise RuntimeError(f"theseus_vocab: the {self._HELD[name]} have been modified by an inplace operation after "
                                   "the loss whose gradients need them")

    def args(self, hidden, weight, loss, row_grad, dhidden, dweight):
        p = lambda t: None if t is None else t.data_ptr()  # noqa: E731
        return LossArgs(self.rows, self.vocab, self.width, self.targets, p(hidden), p(weight),
                        max(hidden.stride(0), self.width), max(weight.stride(0), self.width),
                        p(self.index), p(self.top_values),
                        0 if self.top_values is None else _DTYPES[self.top_values.dtype], _REDUCTIONS[self.reduction],
                        p(self.teacher_lse), p(self.row_weight), self.ignore_index, self.temperature, p(loss), p(row_grad),
                        p(dhidden), p(dweight), self.piece_rows, None, 0)

    def run(self, hidden, weight, loss=None, row_grad=None, dhidden=None, dweight=None, kept=None):
        """``kept`` None: the whole call; True: the forward, returning what it keeps for the gradients
        (None where that is too much); a tensor: the gradients from what the forward kept."""
        lib = _lib()
        a = self.args(hidden, weight, loss, row_grad, dhidden, dweight)
        with torch.cuda.device(self.device):
            if kept is True:
                nbytes = int(lib.theseus_vocab_loss_kept_size(ctypes.byref(a)))
                kept = torch.empty(nbytes, dtype=torch.uint8, device=self.device) if nbytes else None
                a.phase = 0 if kept is None else 1
            elif kept is not None:
                a.phase = 2
            a.kept = None if kept is None else kept.data_ptr()
            nbytes = int(lib.theseus_vocab_loss_workspace_size(ctypes.byref(a)))
            ws = torch.empty(nbytes, dtype=torch.uint8, device=self.device)
            _check(lib.theseus_vocab_loss(ctypes.byref(a), ws.data_ptr(), nbytes, _stream(self.device)))
        return kept

    def new_loss(self):
        return torch.empty(self.rows if self.reduction == "none" else (), dtype=torch.float32, device=self.device)


class _Loss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, hidden, weight, *targets_and_constants):
        # (a trace replays this with tensors that nothing else has looked at)
        hidden, weight, *targets = _laid_out(hidden, weight, *targets_and_constants[:4])
        call = _Call(hidden, weight, *targets, *targets_and_constants[4:])
        loss = call.new_loss()
        need_h, need_w = ctx.needs_input_grad[:2]
        ctx.call, ctx.made, ctx.kept = call, None, None
        if call.reduction == "none":
            ctx.kept = call.run(hidden, weight, loss, kept=True if need_h or need_w else None)
        else:
            ctx.made = _Loss._like(hidden, need_h), _Loss._like(weight, need_w)
            call.run(hidden, weight, loss, None, *ctx.made)
        ctx.save_for_backward(hidden, weight)
        call.hold()
        return loss

    @staticmethod
    def backward(ctx, grad):
        with torch.no_grad():
            made = _Loss._gradients(ctx, grad.float().contiguous())
        if torch.is_grad_enabled():  # (create_graph: a later derivative through these raises)
            made = torch._C._functions.DelayedError("theseus_vocab: the losses are differentiable once", 2)(
                *(x if x is None else x.requires_grad_() for x in made))
        return (*made, *(None,) * 8)

    @staticmethod
    def _like(x, wanted):
        return torch.empty(x.shape, dtype=x.dtype, device=x.device) if wanted else None

    @staticmethod
    def _gradients(ctx, grad):
        call, made, kept = ctx.call, ctx.made, ctx.kept
        ctx.made = ctx.kept = None
        if made is None:
            hidden, weight = ctx.saved_tensors
            need_h, need_w = ctx.needs_input_grad[:2]
            made = _Loss._like(hidden, need_h), _Loss._like(weight, need_w)
            if kept is None:  # (with exponentials, their targets were kept too)
                call.unchanged()
            call.run(hidden, weight, None, grad if call.reduction == "none" else None, *made, kept=kept)
        if call.reduction != "none":
            xy = [v for x in made for v in ((None, 0) if x is None else (x.data_ptr(), x.numel()))]
            with torch.cuda.device(call.device):
                _check(_lib().theseus_vocab_scale(*xy, grad.data_ptr(), _stream(call.device)))
        return made


def _rows(x, name, rows, device, dtypes, tail=()):
    """x [..., *tail] as contiguous [rows, *tail] on the device."""
    if x.dtype not in dtypes:
        raise TypeError(f"theseus_vocab: {name} must be {' or '.join(str(d).replace('torch.', '') for d in dtypes)}, got {x.dtype}")
    if x.device != device:
        raise ValueError(f"theseus_vocab: {name} must be on {device}, got {x.device}")
    if x.shape != rows + tail:
        raise ValueError(f"theseus_vocab: {name} must have shape {list(rows + tail)}, got {list(x.shape)}")
    if len(rows) != 1:
        x = x.reshape(math.prod(rows), *tail)
    return (x.detach() if x.requires_grad else x).contiguous()


def _matrix(x):
    """[n][d] with unit stride along d and rows apart (a strided view's rows are read in place)."""
    if x.stride(1) == 1 and x.stride(0) >= x.shape[1] or x.shape[0] == 1 and x.stride(1) == 1:
        return x
    return x.contiguous()


def _laid_out(hidden, weight, index, top_values, teacher_lse, row_weight):
    """A loss's tensors, checked: hidden [M][D] and weight [V][D] with rows apart, the targets contiguous."""
    if not (hidden.is_cuda and weight.is_cuda):
        raise ValueError("theseus_vocab: hidden and weight must be CUDA tensors")
    shape, size, device = hidden.shape, weight.shape, hidden.device
    if len(shape) < 1 or len(size) != 2 or shape[-1] != size[1] or size[0] < 1 or size[1] < 1:
        raise ValueError(f"theseus_vocab: expected hidden [..., D] and weight [V, D], got {list(shape)} and {list(size)}")
    if size[0] > 1 << 22 or size[1] > 1 << 17 or hidden.numel() > size[1] << 30:
        raise ValueError("theseus_vocab: at most 2^22 words, a width of 2^17 and 2^30 tokens, got "
                         f"hidden {list(shape)} and weight {list(size)}")
    if weight.device != device:
        raise ValueError(f"theseus_vocab: weight must be on {device}, got {weight.device}")
    if hidden.dtype != torch.bfloat16 or weight.dtype != torch.bfloat16:
        raise TypeError(f"theseus_vocab: hidden and weight must be bfloat16 (or cast by autocast), got {hidden.dtype} and {weight.dtype}")
    tokens = shape[:-1]
    index = _rows(index, "labels" if top_values is None else "top_indices", tokens, device, (torch.int64,),
                  () if top_values is None else (index.shape[-1] if index.dim() else 0,))
    if top_values is not None:
        k = index.shape[-1]
        if not 1 <= k <= MAX_TOP:
            raise ValueError(f"theseus_vocab: 1 to {MAX_TOP} top logits per token, got {k}")
        top_values = _rows(top_values, "top_values", tokens, device, tuple(_DTYPES), (k,))
    if teacher_lse is not None:
        teacher_lse = _rows(teacher_lse, "teacher_lse", tokens, device, (torch.float32,))
    if row_weight is not None:
        row_weight = _rows(row_weight, "token_weight", tokens, device, (torch.float32,))
    h, w = _matrix(hidden if len(tokens) == 1 else hidden.reshape(math.prod(tokens), shape[-1])), _matrix(weight)
    if w.stride(0) > MAX_STRIDE:
        w = w.contiguous()
    return h, w, index, top_values, teacher_lse, row_weight


def _loss(hidden, weight, index, top_values, teacher_lse, row_weight, ignore_index, temperature, reduction, piece_rows):
    if reduction not in _REDUCTIONS:
        raise ValueError(f"theseus_vocab: unknown reduction {reduction!r} (none, sum or mean)")
    if not temperature > 0 or temperature == float("inf"):
        raise ValueError(f"theseus_vocab: temperature must be positive, got {temperature}")
    if piece_rows < 0:
        raise ValueError(f"theseus_vocab: piece_rows must not be negative, got {piece_rows}")
    if torch.is_autocast_enabled("cuda") and hidden.is_cuda and weight.is_cuda:
        dt = torch.get_autocast_dtype("cuda")
        hidden, weight = hidden.to(dt), weight.to(dt)
    h, w, *targets = _laid_out(hidden, weight, index, top_values, teacher_lse, row_weight)
    native = _native(h, w)
    if native is not None:
        loss = native.vocab_loss(h, w, *targets, ignore_index, temperature, _REDUCTIONS[reduction], piece_rows)
        return loss.reshape(hidden.shape[:-1]) if reduction == "none" and hidden.dim() != 2 else loss
    constants = ignore_index, float(temperature), reduction, piece_rows
    if _direct(h, w, *targets):
        call = _Call(h, w, *targets, *constants)
        loss = call.new_loss()
        call.run(h, w, loss)
    else:
        loss = _Loss.apply(h, w, *targets, *constants)
    return loss.reshape(hidden.shape[:-1]) if reduction == "none" else loss


def linear_cross_entropy(hidden, weight, labels, *, ignore_index=-100, reduction="mean", piece_rows=0):
    """Softmax cross entropy of ``hidden @ weight.T`` without the logits.

    hidden [..., D], weight [V, D] bfloat16, labels [...] int64.  Returns float32: each token's
    -log p(label) (reduction "none", shape [...]), their sum, or their mean over the tokens whose
    label is not ``ignore_index`` (0 where there is none).  A label outside the vocabulary makes
    its loss NaN.  ``piece_rows``: tokens whose probabilities the gradients hold at a time
    (0: as many as 2 GiB take)."""
    return _loss(hidden, weight, labels, None, None, None, int(ignore_index), 1.0, reduction, int(piece_rows))


def linear_top_distillation(hidden, weight, top_values, top_indices, *, temperature=1.0, teacher_lse=None,
                            token_weight=None, reduction="mean", piece_rows=0):
    """T^2 sum_k q_k (log q_k - log p_k): the divergence of p = softmax(hidden @ weight.T / T)
    from a teacher's top logits, without the student's logits.

    top_values [..., K] (bfloat16 or float32 logits) and top_indices [..., K] int64, K <= 256, as
    ``top_logits`` gives them; -inf entries are left out, equal indices add up.  q is the
    teacher's softmax over the K, or with ``teacher_lse`` [...] (``top_logits``' third result at
    the same temperature) the teacher's own probabilities, what lies outside the K left out.
    token_weight [...] float32 multiplies the tokens' losses (0: the token adds nothing).
    Returns float32: the tokens' losses (reduction "none"), their sum, or the sum over the sum of
    the weights ("mean"; 0 where that is 0)."""
    return _loss(hidden, weight, top_indices, top_values, teacher_lse, token_weight, -100, temperature, reduction,
                 int(piece_rows))


class _Top(torch.autograd.Function):
    """What a trace runs again (its tensors checked and laid out here once more)."""

    @staticmethod
    def forward(ctx, x, k, temperature):
        out = _top(_matrix(_top_checked(x, k)), k, temperature)
        ctx.mark_non_differentiable(*out)
        return out


def _top(x, k, temperature):
    """The C call for x [M][V], rows apart."""
    (n, V), dt, dev = x.shape, _DTYPES[x.dtype], x.device
    values = torch.empty((n, k), dtype=x.dtype, device=dev)
    indices = torch.empty((n, k), dtype=torch.int64, device=dev)
    lse = torch.empty(n, dtype=torch.float32, device=dev)
    lib = _lib()
    with torch.cuda.device(dev):
        nbytes = int(lib.theseus_vocab_top_workspace_size(n, V, k, dt))
        ws = torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None
        _check(lib.theseus_vocab_top(n, V, k, dt, temperature, x.data_ptr(), max(x.stride(0), V), values.data_ptr(),
                                     indices.data_ptr(), lse.data_ptr(), None if ws is None else ws.data_ptr(), nbytes,
                                     _stream(dev)))
    return values, indices, lse


def _top_checked(logits, k):
    if not logits.is_cuda:
        raise ValueError("theseus_vocab: logits must be a CUDA tensor")
    if logits.dtype not in _DTYPES:
        raise TypeError(f"theseus_vocab: logits must be bfloat16 or float32, got {logits.dtype}")
    if logits.dim() < 1 or not 1 <= k <= min(logits.shape[-1], MAX_TOP):
        raise ValueError(f"theseus_vocab: k must be in 1..min(V, {MAX_TOP}), got {k} for logits {list(logits.shape)}")
    if logits.shape[-1] > 1 << 30:
        raise ValueError(f"theseus_vocab: at most 2^30 logits in a row, got {list(logits.shape)}")
    return logits


@torch.no_grad()
def top_logits(logits, k, *, temperature=1.0):
    """The k largest logits of each row: (values [..., k] in the logits' type, indices [..., k]
    int64, lse [...] float32), largest first, equal ones by the lowest index, NaN above every
    number; lse = logsumexp(logits / temperature).

    logits [..., V] bfloat16 or float32 (rows may lie apart: a slice of a wider tensor is read in
    place), 1 <= k <= min(V, 256).  Not differentiable."""
    _top_checked(logits, k)
    if not temperature > 0 or temperature == float("inf"):
        raise ValueError(f"theseus_vocab: temperature must be positive, got {temperature}")
    V, rows = logits.shape[-1], logits.shape[:-1]
    x = _matrix(logits.detach().reshape(math.prod(rows), V))
    native = _native(x)
    if native is not None:
        out = native.vocab_top(x, k, float(temperature))
    else:
        out = (_top if _direct(x) else _Top.apply)(x, k, float(temperature))
    if len(rows) == 1:
        return out
    values, indices, lse = out
    return values.reshape(*rows, k), indices.reshape(*rows, k), lse.reshape(rows)
