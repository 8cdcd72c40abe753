"""Row operators next to `log_softmax`: layer normalisation of frame embeddings, the loss of a head's logits against frame labels,
and labels drawn from the logits -- with the gradients by which the model in front of the aligner is trained.

    embeddings -> layer_norm -> (projection) -> logits -> align_batch / sample_labels -> labels -> label_loss -> gradients

Every operator takes rows [B, T, C] (or [B, C], one row per sequence; any leading shape without `lengths`) of float32, float16 or
bfloat16 on the GPU, with any strides as long as the last one is 1 (others are copied), and `lengths` [B]: rows behind
an utterance's length are not read and come out as 0 (labels: -1).  The kernels are those behind include/bfa.h; the work is
stream-ordered on the current stream of the tensors' device and nothing synchronises.

A backward pass may be captured into a graph like the forward pass.  PyTorch ends the process when `backward()` accumulates into the
`.grad` of a leaf inside a capture while a graph built outside the capture from the same leaf is alive: capture with
`torch.autograd.grad`, or call `layer_norm_backward` / `label_loss_and_grad`, which build no graph."""
import ctypes

import torch
import torch.autograd.forward_ad as _forward_ad

from . import _lib
from .forced_alignment import HostLens, _as_i32

_DTYPES = {torch.float32: _lib.DTYPE_F32, torch.float16: _lib.DTYPE_F16, torch.bfloat16: _lib.DTYPE_BF16}
_REDUCTIONS = {"none": _lib.LOSS_NONE, "sum": _lib.LOSS_SUM, "mean": _lib.LOSS_MEAN}


def _check_rows(x, what):
    if not (isinstance(x, torch.Tensor) and x.is_cuda):
        raise RuntimeError(f"{what} runs on the GPU only: pass a device tensor (there is no CPU fallback)")
    if x.dtype not in _DTYPES:
        raise TypeError(f"{what}: rows must be float32, float16 or bfloat16, not {x.dtype}")
    if x.dim() < 1:
        raise ValueError(f"{what}: rows need at least one dimension")


def _shape_of(x, lengths, what):
    """(B, T) of rows [B, T, C], [B, C] (T = 1) or, without lengths, of any leading shape"""
    lead = x.shape[:-1]
    if len(lead) == 2:
        B, T = lead
    elif len(lead) == 1:
        B, T = lead[0], 1
    elif lengths is not None:
        raise ValueError(f"{what}: lengths go with rows [B, T, C] or [B, C], not {tuple(x.shape)}")
    else:
        B, T = lead.numel(), 1
    if B * T >= 1 << 31:
        raise ValueError(f"{what}: at most 2^31 - 1 rows")
    if x.shape[-1] > 1 << 30:
        raise ValueError(f"{what}: rows of at most 2^30 elements")
    return B, T


def _rows(x, B, T):
    """(a tensor that holds the rows, the bfa_rows that describes it)"""
    if x.dim() not in (2, 3):
        x = x.reshape(B, T, x.shape[-1])
    if x.stride(-1) != 1 and x.shape[-1] > 1:
        x = x.contiguous()
    sT = x.stride(1) if x.dim() == 3 else 0
    return x, _lib.BfaRows(x.data_ptr(), _DTYPES[x.dtype], x.stride(0), sT)


def _lengths(lengths, B, dev, what):
    if lengths is None:
        return None
    if isinstance(lengths, torch.Tensor) and lengths.dtype == torch.int32 and lengths.device == dev and lengths.shape == (B,):
        return lengths.contiguous()
    n = len(lengths) if not isinstance(lengths, torch.Tensor) else lengths.numel()
    if n != B or (isinstance(lengths, torch.Tensor) and lengths.dim() != 1):
        raise ValueError(f"{what}: lengths must have one entry per utterance ({B})")
    return _as_i32(lengths, dev)


def _per_row(t, shape, dtype, dev, what, name):
    """a [B, T] companion of the rows on their device"""
    if isinstance(t, HostLens) or not isinstance(t, torch.Tensor):
        t = torch.as_tensor(t)
    if tuple(t.shape) != tuple(shape):
        raise ValueError(f"{what}: {name} must have the shape {tuple(shape)} of the rows, not {tuple(t.shape)}")
    if t.is_cuda and t.device != dev:
        raise ValueError(f"{what}: {name} is on {t.device}, the rows on {dev}")
    if dtype == torch.int32 and (t.is_floating_point() or t.is_complex()):
        raise TypeError(f"{what}: {name} must be whole numbers")
    if t.dtype != dtype or t.device != dev:
        t = t.to(device=dev, dtype=dtype)
    return t.contiguous()


def _ptr(t):
    return None if t is None else t.data_ptr()


# the current stream's handle without the object around it, where this torch has that
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda index: torch.cuda.current_stream(index).cuda_stream)


def _call(dev):
    # (the C entries work on their handle's device, whatever the current one is)
    return _lib.lib(), _lib.handle(dev.index), _raw_stream(dev.index)


def _tangent(t):
    return _forward_ad.unpack_dual(t).tangent if _forward_ad._current_level >= 0 and isinstance(t, torch.Tensor) else None


def _wants_graph(*tensors):
    """whether a call has to go through its autograd function: an input requires a gradient, or forward-mode differentiation is on
    (the functions have no rule for it, and torch says so where an input has a tangent)"""
    if _forward_ad._current_level >= 0:
        return True
    return torch.is_grad_enabled() and any(getattr(t, "requires_grad", False) for t in tensors)


def _backward_of(fn):
    """fn(ctx, *gradients) as a backward pass that cannot be differentiated again; what that takes is spent only when a graph of the
    gradients is built"""
    once = torch.autograd.function.once_differentiable(fn)
    return staticmethod(lambda ctx, *grads: (once if torch.is_grad_enabled() else fn)(ctx, *grads))


# ---- layer normalisation ---------------------------------------------------------------------------------------------------

def _norm_params(x, weight, bias):
    wdt = None
    for name, t in (("weight", weight), ("bias", bias)):
        if t is None:
            continue
        if not isinstance(t, torch.Tensor) or t.dtype not in _DTYPES:
            raise TypeError(f"layer_norm: {name} must be a float32, float16 or bfloat16 tensor")
        if t.device != x.device or tuple(t.shape) != (x.shape[-1],):
            raise ValueError(f"layer_norm: {name} must have shape ({x.shape[-1]},) on {x.device}")
        if wdt is not None and t.dtype != wdt:
            raise TypeError("layer_norm: weight and bias must have one type")
        wdt = t.dtype
    return _lib.DTYPE_F32 if wdt is None else _DTYPES[wdt]


def layer_norm_forward(x, weight=None, bias=None, eps=1e-5, lengths=None, statistics=True):
    """(y, mean, rstd): y as `layer_norm` gives it (without a gradient of either mode), the rows' statistics float32 of the leading shape (None,
    None without `statistics`) as `layer_norm_backward` takes them."""
    _check_rows(x, "layer_norm")
    B, T = _shape_of(x, lengths, "layer_norm")
    wt = _norm_params(x, weight, bias)
    if not eps >= 0:
        raise ValueError("layer_norm: eps must not be negative")
    dev, C = x.device, x.shape[-1]
    lens = _lengths(lengths, B, dev, "layer_norm")
    weight = None if weight is None else weight.contiguous()
    bias = None if bias is None else bias.contiguous()
    y = torch.empty(x.shape, dtype=x.dtype, device=dev)
    mean = torch.empty(x.shape[:-1], dtype=torch.float32, device=dev) if statistics else None
    rstd = torch.empty_like(mean) if statistics else None
    keep, rx = _rows(x, B, T)
    ry = _lib.BfaRows(y.data_ptr(), rx.dtype, T * C, C)
    L, h, stream = _call(dev)
    rc = L.bfa_layer_norm(h, ctypes.byref(rx), B, T, C, _ptr(lens), _ptr(weight), _ptr(bias), wt, eps, ctypes.byref(ry),
                          _ptr(mean), _ptr(rstd), stream)
    _lib.check(rc, h, "bfa_layer_norm")
    return y, mean, rstd


def layer_norm_backward(grad, x, mean, rstd, weight=None, lengths=None, param_dtype=None, need=(True, True, True)):
    """(dx, dweight, dbias) of `layer_norm` for the gradient of its result, with the statistics of `layer_norm_forward`; entries
    that `need` does not ask for are None.  dweight and dbias have the weight's type, or `param_dtype` (default float32) without
    a weight."""
    _check_rows(x, "layer_norm_backward")
    B, T = _shape_of(x, lengths, "layer_norm_backward")
    _norm_params(x, weight, None)
    dev, C = x.device, x.shape[-1]
    if not isinstance(grad, torch.Tensor) or grad.device != dev or grad.dtype != x.dtype or grad.shape != x.shape:
        raise ValueError("layer_norm_backward: grad must match x in shape, type and device")
    for name, t in (("mean", mean), ("rstd", rstd)):
        if not isinstance(t, torch.Tensor) or t.device != dev or t.dtype != torch.float32 or t.shape != x.shape[:-1]:
            raise ValueError(f"layer_norm_backward: {name} must be float32 of shape {tuple(x.shape[:-1])} on {dev}")
    pdt = weight.dtype if weight is not None else (param_dtype or torch.float32)
    if pdt not in _DTYPES:
        raise TypeError("layer_norm_backward: param_dtype must be float32, float16 or bfloat16")
    return _norm_backward(grad, x, mean.contiguous(), rstd.contiguous(), weight, _lengths(lengths, B, dev, "layer_norm_backward"), pdt, need, B, T)


def _norm_backward(grad, x, mean, rstd, weight, lens, pdt, need, B, T):
    dev, C = x.device, x.shape[-1]
    weight = None if weight is None else weight.contiguous()
    dx = torch.empty(x.shape, dtype=x.dtype, device=dev) if need[0] else None
    make = torch.zeros if B * T == 0 else torch.empty
    dw = make(C, dtype=pdt, device=dev) if need[1] else None
    db = make(C, dtype=pdt, device=dev) if need[2] else None
    kx, rx = _rows(x, B, T)
    kg, rg = _rows(grad, B, T)
    rdx = _lib.BfaRows(dx.data_ptr(), rx.dtype, T * C, C) if dx is not None else None
    L, h, stream = _call(dev)
    nbytes = L.bfa_layer_norm_workspace_bytes(B, T, C) if need[1] or need[2] else 0
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None
    rc = L.bfa_layer_norm_backward(h, ctypes.byref(rg), ctypes.byref(rx), B, T, C, _ptr(lens), _ptr(weight), _DTYPES[pdt],
                                   _ptr(mean), _ptr(rstd), ctypes.byref(rdx) if rdx is not None else None, _ptr(dw), _ptr(db),
                                   _ptr(ws), nbytes, stream)
    _lib.check(rc, h, "bfa_layer_norm_backward")
    return dx, dw, db


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps, lengths):
        y, mean, rstd = layer_norm_forward(x, weight, bias, eps, lengths)
        ctx.save_for_backward(x, weight, mean, rstd, lengths)
        ctx.bias_dtype = None if bias is None else bias.dtype
        return y

    @_backward_of
    def backward(ctx, grad):
        x, weight, mean, rstd, lens = ctx.saved_tensors
        B, T = _shape_of(x, lens, "layer_norm")
        pdt = weight.dtype if weight is not None else (ctx.bias_dtype or torch.float32)
        return (*_norm_backward(grad, x, mean, rstd, weight, lens, pdt, ctx.needs_input_grad[:3], B, T), None, None)


def layer_norm(x, weight=None, bias=None, eps=1e-5, lengths=None):
    """(x - mean) / sqrt(var + eps) * weight + bias over the last dimension, differentiable in x, weight and bias.  weight and bias
    [C] have one type, the rows' or another of the three; mean, variance and all sums are float32."""
    _check_rows(x, "layer_norm")
    if _wants_graph(x, weight, bias):
        B, _ = _shape_of(x, lengths, "layer_norm")
        return _LayerNorm.apply(x, weight, bias, eps, _lengths(lengths, B, x.device, "layer_norm"))
    return layer_norm_forward(x, weight, bias, eps, lengths, statistics=False)[0]


# ---- the loss of logits against labels -------------------------------------------------------------------------------------

def _loss_args(logits, labels, weights, lengths, reduction):
    _check_rows(logits, "label_loss")
    if reduction not in _REDUCTIONS:
        raise ValueError(f"label_loss: reduction must be 'none', 'sum' or 'mean', not {reduction!r}")
    B, T = _shape_of(logits, lengths, "label_loss")
    shape, dev = logits.shape[:-1], logits.device
    labels = _per_row(labels, shape, torch.int32, dev, "label_loss", "labels")
    weights = None if weights is None else _per_row(weights, shape, torch.float32, dev, "label_loss", "weights").detach()
    return labels, weights, _lengths(lengths, B, dev, "label_loss")


def _loss_call(logits, labels, weights, lens, reduction, want_loss, want_grad, scale=1.0, upstream=None):
    B, T = _shape_of(logits, lens, "label_loss")
    dev, C, red = logits.device, logits.shape[-1], _REDUCTIONS[reduction]
    make = torch.zeros if C == 0 else torch.empty
    loss = make(logits.shape[:-1] if red == _lib.LOSS_NONE else (), dtype=torch.float32, device=dev) if want_loss else None
    grad = torch.empty(logits.shape, dtype=logits.dtype, device=dev) if want_grad else None
    keep, rz = _rows(logits, B, T)
    rg = _lib.BfaRows(grad.data_ptr(), rz.dtype, T * C, C) if want_grad else None
    L, h, stream = _call(dev)
    nbytes = L.bfa_label_loss_workspace_bytes(B, T, C) if red != _lib.LOSS_NONE else 0
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None
    rc = L.bfa_label_loss(h, ctypes.byref(rz), B, T, C, _ptr(lens), labels.data_ptr(), _ptr(weights), red, scale, _ptr(upstream),
                          _ptr(loss), ctypes.byref(rg) if want_grad else None, _ptr(ws), nbytes, stream)
    _lib.check(rc, h, "bfa_label_loss")
    return loss, grad


class _LabelLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, labels, weights, lens, reduction):
        ctx.save_for_backward(logits, labels, weights, lens)
        ctx.reduction = reduction
        return _loss_call(logits, labels, weights, lens, reduction, True, False)[0]

    @_backward_of
    def backward(ctx, upstream):
        logits, labels, weights, lens = ctx.saved_tensors
        upstream = upstream.to(torch.float32).contiguous()
        return _loss_call(logits, labels, weights, lens, ctx.reduction, False, True, upstream=upstream)[1], None, None, None, None


def label_loss(logits, labels, weights=None, lengths=None, reduction="mean"):
    """Weighted cross entropy -weight * log softmax(logits)[label] of every row, float32, differentiable in the logits (not in the
    weights: those that require a gradient are refused).  Rows with a negative label (an alignment's -1) or weight 0 and rows behind
    `lengths` give 0; a label >= C gives NaN (labels are taken as int32).  reduction: 'none' (one per row), 'sum', or 'mean' (divided
    by the sum of the weights of the rows that count; 0 where that is 0)."""
    if (torch.is_grad_enabled() and getattr(weights, "requires_grad", False)) or _tangent(weights) is not None:
        raise ValueError("label_loss: no gradient goes to the weights: pass weights.detach()")
    labels, weights, lens = _loss_args(logits, labels, weights, lengths, reduction)
    if _wants_graph(logits):
        return _LabelLoss.apply(logits, labels, weights, lens, reduction)
    return _loss_call(logits, labels, weights, lens, reduction, True, False)[0]


def label_loss_and_grad(logits, labels, weights=None, lengths=None, reduction="mean", grad_scale=1.0):
    """(loss, gradient of grad_scale * loss in the logits) in one pass over them, for training steps that know the factor of the
    loss beforehand: the logits are read once, where `label_loss` and its backward pass read them twice.  With 'none' the
    gradient is that of grad_scale * (the sum of the rows' losses)."""
    labels, weights, lens = _loss_args(logits, labels, weights, lengths, reduction)
    return _loss_call(logits, labels, weights, lens, reduction, True, True, scale=float(grad_scale))


# ---- labels drawn from logits ----------------------------------------------------------------------------------------------

def sample_labels(logits, uniform, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, lengths=None):
    """(labels int32, logp float32) of the rows' leading shape: one class per row from softmax(logits / temperature), kept to the
    `top_k` most probable classes (0: all), of those to the fewest that hold `top_p` of their probability, and to classes with at least
    `min_p` of the greatest probability; logp is the logarithm of the drawn class's probability among the kept ones (without a
    gradient; up to 512 classes from a float32 sum, good to about 2^-22).

    `uniform`: one number in [0, 1) per row; the label is the lowest class up to which, in the order of the classes, more than that share
    of the kept probability lies, so the same numbers give the same labels.  The parameters are numbers, or tensors [B] with
    one per utterance (sequence), or one number in a tensor; they are taken as float32.  temperature 0 takes the most probable class (of equals the lowest).
    -inf masks a class and NaN counts as -inf; rows with nothing left, and rows behind `lengths`, give label -1 and logp 0."""
    _check_rows(logits, "sample_labels")
    B, T = _shape_of(logits, lengths, "sample_labels")
    dev, C = logits.device, logits.shape[-1]
    uniform = _per_row(uniform, logits.shape[:-1], torch.float32, dev, "sample_labels", "uniform")
    lens = _lengths(lengths, B, dev, "sample_labels")
    p = _lib.BfaSampleParams()
    keep = []
    for name, value, dt in (("temperature", temperature, torch.float32), ("top_k", top_k, torch.int32),
                            ("top_p", top_p, torch.float32), ("min_p", min_p, torch.float32)):
        if isinstance(value, torch.Tensor) and (value.dim() > 0 or value.is_cuda):  # (one number on the device is not read here)
            if value.dtype == torch.int64 and dt == torch.int32:
                value = value.clamp(0, 0x7fffffff)  # (as a number is: a value of 33 bits does not come out as its low 32)
            value = _per_row(value if value.dim() > 0 else value.expand(B), (B,), dt, dev, "sample_labels", name)
            keep.append(value)
            setattr(p, name + "_B", value.data_ptr())
            continue
        if name == "temperature" and not value >= 0:
            raise ValueError("sample_labels: temperature must not be negative")
        if name == "top_p" and not 0 < value:
            raise ValueError("sample_labels: top_p must be positive")
        if name == "min_p" and not 0 <= value <= 1:
            raise ValueError("sample_labels: min_p must be in [0, 1]")
        setattr(p, name, min(max(int(value), 0), 0x7fffffff) if name == "top_k" else float(value))
    make = torch.zeros if C == 0 else torch.empty
    labels = make(logits.shape[:-1], dtype=torch.int32, device=dev)
    logp = make(logits.shape[:-1], dtype=torch.float32, device=dev)
    if C == 0:
        return labels.fill_(-1), logp
    kz, rz = _rows(logits.detach(), B, T)
    L, h, stream = _call(dev)
    rc = L.bfa_sample_labels(h, ctypes.byref(rz), B, T, C, _ptr(lens), uniform.data_ptr(), ctypes.byref(p), labels.data_ptr(),
                             logp.data_ptr(), stream)
    _lib.check(rc, h, "bfa_sample_labels")
    return labels, logp
