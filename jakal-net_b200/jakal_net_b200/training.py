"""Training-step operators around the propagation / transition operators: the layer norm of an
apply step, the loss over the query head's vocabulary, and the clipping of the gradients.

A Jakal-Net training step applies every operator's delta to its layer as
``LayerNorm(x + scale * delta)`` (progressive_b_example.py:71-99, 282-294), ends in a softmax
cross entropy over the vocabulary and clips the global gradient norm before the optimizer.
The functions come in two forms, as the other training operators of this package do:

* ``*_cuda`` entry points over plain tensors (no autograd graph): ``layer_norm_forward_cuda``,
  ``layer_norm_backward_cuda``, ``cross_entropy_forward_cuda``, ``cross_entropy_backward_cuda``,
  ``cross_entropy_with_grad_cuda``, ``grad_norm``, ``clip_grad_norm_``;
* ``layer_norm`` and ``cross_entropy``, which autograd differentiates through those.

Inputs are CUDA tensors in f32, bf16 or f16, rows contiguous inside (other layouts are copied
first); arithmetic and sums are f32 or wider whatever autocast says, and a result keeps its
input's type. Everything runs on the current stream, allocates through torch and reads nothing
back, so calls can be captured into a CUDA graph. Results are the same from run to run.
"""
from __future__ import annotations

import array
import math
import operator
from typing import Iterable, Optional, Union

import torch
from torch import Tensor

from . import _lib
from ._lib import check, load

__all__ = [
    "layer_norm",
    "layer_norm_forward_cuda",
    "layer_norm_backward_cuda",
    "cross_entropy",
    "cross_entropy_forward_cuda",
    "cross_entropy_backward_cuda",
    "cross_entropy_with_grad_cuda",
    "grad_norm",
    "clip_grad_norm_",
]

_LIBRARY = load()
_DTYPE_CODE = {torch.float32: _lib.JK_F32, torch.bfloat16: _lib.JK_BF16, torch.float16: _lib.JK_F16}
_current_device, _raw_stream = torch._C._cuda_getDevice, torch._C._cuda_getCurrentRawStream
_REDUCTION = {"none": _lib.JK_REDUCE_NONE, "mean": _lib.JK_REDUCE_MEAN, "sum": _lib.JK_REDUCE_SUM}


# ----------------------------------------------------------------------------- helpers
def _check_input(name: str, t: Tensor) -> int:
    """The dtype code of a CUDA float tensor; anything else raises."""
    if not isinstance(t, Tensor):
        raise TypeError(f"{name} must be a tensor")
    code = _DTYPE_CODE.get(t.dtype)
    if code is None or not t.is_cuda:
        if not t.is_cuda:
            raise RuntimeError(f"{name} must be a CUDA tensor in the b200_sm100a backend (got {t.device}).")
        raise RuntimeError(f"{name}: unsupported dtype {t.dtype}")
    return code


def _same(name: str, t: Tensor, like: Tensor) -> None:
    """t has like's device, dtype and shape."""
    if not isinstance(t, Tensor):
        raise TypeError(f"{name} must be a tensor")
    if t.get_device() != like.get_device():
        raise RuntimeError(f"{name} is on {t.device}, expected {like.device}")
    if t.dtype != like.dtype:
        raise RuntimeError(f"{name} has dtype {t.dtype}, expected {like.dtype}")
    if t.shape != like.shape:
        raise ValueError(f"{name} has shape {tuple(t.shape)}, expected {tuple(like.shape)}")


def _rows(t: Tensor) -> tuple[Tensor, int]:
    """(t, elements from one row to the next), rows along the last dim: t itself where its rows
    are contiguous inside and equally spaced (a slice of wider rows, an expanded row), else a
    contiguous copy."""
    if t.is_contiguous():
        return t, t.shape[-1]
    t = t.detach()
    if t.stride(-1) == 1 or t.shape[-1] == 1:
        try:
            return t, t.view(-1, t.shape[-1]).stride(0)
        except RuntimeError:  # leading dims that no single stride spans
            pass
    return t.contiguous(), t.shape[-1]


def _written(tensors: list[Tensor]) -> None:
    """Tells autograd that the kernels wrote over these tensors (a value kept for a backward
    pass is then seen to be stale); inference tensors, which have no version, may be among them."""
    if tensors:
        torch.autograd.graph.increment_version(tensors)


def _call(fn, where: str, device: int, *args) -> None:
    """fn(*args, stream) on the device's current stream, with the device current; raises on a
    status that is not 0."""
    if _current_device() == device:
        status = fn(*args, _raw_stream(device))
    else:
        with torch.cuda.device(device):
            status = fn(*args, _raw_stream(device))
    if status:
        check(status, where)


def _param(name: str, p: Tensor, device: int, dim: int) -> tuple[Tensor, int]:
    """(a contiguous [dim] parameter on the device, its dtype code)"""
    code = _check_input(name, p)
    if p.get_device() != device:
        raise RuntimeError(f"{name} is on {p.device}, expected cuda:{device}")
    if p.dim() != 1 or p.numel() != dim:
        raise ValueError(f"{name} has shape {tuple(p.shape)}, expected {(dim,)}")
    return (p if p.is_contiguous() else p.detach().contiguous()), code


def _empty_like(t: Tensor) -> Tensor:
    """An uninitialised contiguous tensor of t's shape, dtype and device."""
    return torch.empty_like(t) if t.is_contiguous() else torch.empty_like(t, memory_format=torch.contiguous_format)


def _empty(shape, dtype: torch.dtype, device: torch.device) -> Tensor:
    """torch.empty, by its quickest way for no and for one dim."""
    n = len(shape)
    if n > 1:
        return torch.empty(shape, dtype=dtype, device=device)
    return torch.empty_strided(shape, (1,) * n, dtype=dtype, device=device)


def _ptr(t: Optional[Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


# ----------------------------------------------------------------------------- layer norm
def layer_norm_forward_cuda(x: Tensor, weight: Optional[Tensor] = None, bias: Optional[Tensor] = None,
                            eps: float = 1e-5, delta: Optional[Tensor] = None, delta_scale: float = 1.0):
    """Layer norm over the last dim of ``sum = x + delta_scale * delta`` (delta None: of x).

    Returns (y, sum, mean, rstd): y and sum in x's dtype and shape (sum is x itself without a
    delta), mean and rstd f32 of x's leading shape, for ``layer_norm_backward_cuda``. y is
    normalised from the sum before it is rounded. delta has x's dtype and shape; weight and bias
    are [dim], of one dtype, x's or another."""
    code = _check_input("x", x)
    if x.dim() == 0:
        raise ValueError("x must have at least one dim")
    dim = x.shape[-1]
    if dim == 0:
        raise ValueError("the normalised dim is empty")
    device, pcode = x.get_device(), code
    weight_at = bias_at = delta_at = sum_at = None
    if weight is not None:
        weight, pcode = _param("weight", weight, device, dim)
        weight_at = weight.data_ptr()
    if bias is not None:
        bias, bcode = _param("bias", bias, device, dim)
        bias_at = bias.data_ptr()
        if weight is not None and bcode != pcode:
            raise RuntimeError(f"weight and bias have different dtypes ({weight.dtype}, {bias.dtype})")
        pcode = bcode
    xr, x_stride = _rows(x)
    y = _empty_like(x)
    total, d_stride = x, 0
    if delta is not None:
        _same("delta", delta, x)
        dr, d_stride = _rows(delta)
        total = torch.empty_like(y)
        delta_at, sum_at = dr.data_ptr(), total.data_ptr()
    mean = _empty(x.shape[:-1], torch.float32, x.device)
    rstd = torch.empty_like(mean)
    _call(_LIBRARY.jk_layer_norm_forward, "jk_layer_norm_forward", device, xr.data_ptr(), x_stride, delta_at, d_stride,
          delta_scale, weight_at, bias_at, pcode, mean.numel(), dim, code, eps, y.data_ptr(), sum_at, mean.data_ptr(),
          rstd.data_ptr())
    return y, total, mean, rstd


def layer_norm_backward_cuda(grad_y: Tensor, sum: Tensor, mean: Tensor, rstd: Tensor, weight: Optional[Tensor] = None,
                             grad_sum: Optional[Tensor] = None, delta_scale: float = 1.0, param_grads: bool = True,
                             param_dtype: Optional[torch.dtype] = None):
    """Backward of ``layer_norm_forward_cuda`` from the sum and statistics that it returned.

    Returns (grad_x, grad_delta, grad_weight, grad_bias). grad_sum is the gradient that reaches
    the sum from its other uses (the residual stream); grad_delta is grad_x itself when
    delta_scale is 1. The parameter gradients have weight's dtype, without a weight param_dtype
    (None: the sum's); param_grads=False returns None for them."""
    code = _check_input("sum", sum)
    if sum.dim() == 0 or sum.shape[-1] == 0:
        raise ValueError("sum must have a last dim that is not empty")
    dim = sum.shape[-1]
    _same("grad_y", grad_y, sum)
    device, pcode = sum.get_device(), code
    weight_at = gs_at = gd_at = gw_at = gb_at = work_at = None
    if weight is not None:
        weight, pcode = _param("weight", weight, device, dim)
        weight_at = weight.data_ptr()
        if param_dtype not in (None, weight.dtype):
            raise RuntimeError(f"param_dtype {param_dtype} is not the weight's dtype {weight.dtype}")
    elif param_dtype is not None:
        pcode = _DTYPE_CODE.get(param_dtype)
        if pcode is None:
            raise RuntimeError(f"param_dtype: unsupported dtype {param_dtype}")
    lead = sum.shape[:-1]
    for name, t in (("mean", mean), ("rstd", rstd)):
        if not isinstance(t, Tensor) or t.dtype != torch.float32 or t.get_device() != device:
            raise RuntimeError(f"{name} must be an f32 tensor on {sum.device}")
        if t.shape != lead:
            raise ValueError(f"{name} has shape {tuple(t.shape)}, expected {tuple(lead)}")
    mean, rstd = mean.contiguous(), rstd.contiguous()
    gy, gy_stride = _rows(grad_y)
    hr, h_stride = _rows(sum)
    gs_stride = 0
    if grad_sum is not None:
        _same("grad_sum", grad_sum, sum)
        gs, gs_stride = _rows(grad_sum)
        gs_at = gs.data_ptr()
    rows = mean.numel()
    grad_x = grad_delta = _empty_like(sum)
    if delta_scale != 1.0:
        grad_delta = torch.empty_like(grad_x)
        gd_at = grad_delta.data_ptr()
    grad_weight = grad_bias = None
    if param_grads:
        grad_weight = torch.empty_like(weight) if weight is not None else sum.new_empty((dim,), dtype=param_dtype)
        grad_bias = torch.empty_like(grad_weight)
        work = _empty((_LIBRARY.jk_layer_norm_backward_workspace(rows, dim),), torch.float32, sum.device)
        gw_at, gb_at, work_at = grad_weight.data_ptr(), grad_bias.data_ptr(), work.data_ptr()
    _call(_LIBRARY.jk_layer_norm_backward, "jk_layer_norm_backward", device, gy.data_ptr(), gy_stride, hr.data_ptr(), h_stride,
          mean.data_ptr(), rstd.data_ptr(), weight_at, pcode, gs_at, gs_stride, delta_scale, rows, dim, code,
          grad_x.data_ptr(), gd_at, gw_at, gb_at, work_at)
    return grad_x, grad_delta, grad_weight, grad_bias


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps, delta, delta_scale):
        y, total, mean, rstd = layer_norm_forward_cuda(x, weight, bias, eps, delta, delta_scale)
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(total, mean, rstd, weight)
        ctx.delta_scale, ctx.has_delta = delta_scale, delta is not None
        ctx.bias_dtype = None if bias is None else bias.dtype
        return (y, total) if delta is not None else y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_y, grad_sum=None):
        total, mean, rstd, weight = ctx.saved_tensors
        need_x, need_w, need_b, _, need_delta, _ = ctx.needs_input_grad
        if grad_y is None and grad_sum is None:
            return (None,) * 6
        if grad_y is None:  # only the residual stream was used: the norm's part is zero
            grad_y = torch.zeros_like(total)
        gx, gd, gw, gb = layer_norm_backward_cuda(grad_y, total, mean, rstd, weight, grad_sum, ctx.delta_scale,
                                                  need_w or need_b, ctx.bias_dtype if weight is None else None)
        return gx if need_x else None, gw if need_w else None, gb if need_b else None, None, gd if need_delta else None, None


def layer_norm(x: Tensor, weight: Optional[Tensor] = None, bias: Optional[Tensor] = None, eps: float = 1e-5,
               delta: Optional[Tensor] = None, delta_scale: float = 1.0):
    """Differentiable layer norm of an apply step: y, or (y, sum) when a delta is given."""
    return _LayerNorm.apply(x, weight, bias, float(eps), delta, float(delta_scale))


# ----------------------------------------------------------------------------- cross entropy
def _loss_inputs(logits: Tensor, targets: Tensor, reduction: str):
    code = _check_input("logits", logits)
    if logits.dim() == 0 or logits.shape[-1] == 0:
        raise ValueError("logits must have a last dim (the vocabulary) that is not empty")
    if not isinstance(targets, Tensor):
        raise TypeError("targets must be a tensor")
    if targets.device != logits.device:
        raise RuntimeError(f"targets are on {targets.device}, expected {logits.device}")
    if targets.dtype not in (torch.int64, torch.int32):
        raise RuntimeError(f"targets: unsupported dtype {targets.dtype} (int64 or int32)")
    if targets.shape != logits.shape[:-1]:
        raise ValueError(f"targets have shape {tuple(targets.shape)}, expected {tuple(logits.shape[:-1])}")
    kind = _REDUCTION.get(reduction)
    if kind is None:
        raise ValueError(f"unknown reduction {reduction!r} (none, mean or sum)")
    if targets.dtype != torch.int64 or not targets.is_contiguous():
        targets = targets.to(torch.int64).contiguous()
    lr, stride = _rows(logits)
    return code, targets, kind, lr, stride


def _grad_like(logits: Tensor, rows: Tensor, stride: int) -> Tensor:
    """An uninitialised gradient whose rows lie against 16-byte blocks as the logits' rows do, where
    those are equally spaced and apart; else a contiguous one. Rows are spaced as the logits' are while
    the padding between them is an eighth of a row at most (a padded vocabulary), else (one position
    of each sequence, a slice of the vocabulary) as closely as that allows.
    (rows, stride): the logits as ``_rows`` has them."""
    shift = logits.data_ptr() % 16
    if logits.is_contiguous() and not shift:
        return torch.empty_like(logits)
    vocab = logits.shape[-1]
    if logits.numel() == 0 or rows.data_ptr() != logits.data_ptr() or stride < vocab:
        return _empty_like(logits)
    size = logits.element_size()
    shift //= size
    n = logits.numel() // vocab
    if stride - vocab <= vocab // 8:
        return logits.new_empty((shift + n * stride,)).as_strided(logits.shape, logits.stride(), shift)
    stride = vocab + (stride - vocab) % (16 // size)
    return logits.new_empty((shift + n * stride,)).as_strided((n, vocab), (stride, 1), shift).view(logits.shape)


def _cross_entropy(logits, targets, ignore_index, label_smoothing, reduction, grad_scale, want_lse=False, want_grad=False,
                   in_place=False):
    """(loss, lse, gradient), the latter two None where they are not asked for; in_place: the gradient
    goes over the logits."""
    code, targets, kind, lr, stride = _loss_inputs(logits, targets, reduction)
    rows, device = targets.numel(), logits.device
    lse = losses = grad = None
    if kind == _lib.JK_REDUCE_NONE:
        loss = losses = _empty(targets.shape, torch.float32, device)
    else:
        loss = _empty((), torch.float32, device)
    if want_lse:
        lse = torch.empty_like(loss) if losses is not None else _empty(targets.shape, torch.float32, device)
    work = _empty((_LIBRARY.jk_cross_entropy_workspace(rows) // 4,), torch.float32, device)
    grad_ptr, grad_stride = None, 0
    if in_place:
        grad_ptr, grad_stride = lr.data_ptr(), stride
    elif want_grad:
        grad = _grad_like(logits, lr, stride)
        grad_ptr, grad_stride = grad.data_ptr(), _rows(grad)[1]
    _call(_LIBRARY.jk_cross_entropy_forward, "jk_cross_entropy_forward", logits.get_device(), lr.data_ptr(), stride,
          targets.data_ptr(), rows, logits.shape[-1], code, ignore_index, label_smoothing, kind, grad_scale, _ptr(losses),
          _ptr(lse), None if losses is not None else loss.data_ptr(), grad_ptr, grad_stride, work.data_ptr())
    return loss, lse, grad


def _cross_entropy_split(logits, targets, ignore_index, label_smoothing, reduction):
    """(loss, log-sums): the latter as two f32 each, [2, *targets.shape], whose sum they are."""
    code, targets, kind, lr, stride = _loss_inputs(logits, targets, reduction)
    rows, device = targets.numel(), logits.device
    lse = torch.empty((2, *targets.shape), dtype=torch.float32, device=device)
    each = kind == _lib.JK_REDUCE_NONE
    loss = _empty(targets.shape if each else (), torch.float32, device)
    work = _empty((_LIBRARY.jk_cross_entropy_workspace(rows) // 4,), torch.float32, device)
    at = loss.data_ptr()
    _call(_LIBRARY.jk_cross_entropy_forward_split, "jk_cross_entropy_forward_split", logits.get_device(), lr.data_ptr(), stride,
          targets.data_ptr(), rows, logits.shape[-1], code, ignore_index, label_smoothing, kind, at if each else None,
          lse.data_ptr(), lse.data_ptr() + 4 * rows, None if each else at, work.data_ptr())
    return loss, lse


def cross_entropy_forward_cuda(logits: Tensor, targets: Tensor, ignore_index: int = -100, label_smoothing: float = 0.0,
                               reduction: str = "mean"):
    """Softmax cross entropy of logits [..., vocab] against int64 (or int32) targets [...].

    Returns (loss, lse): loss f32, a scalar for reduction "mean" (over the targets that are not
    ignore_index) or "sum", of targets' shape for "none"; lse f32 of targets' shape, the rows'
    log-sum-exp, which ``cross_entropy_backward_cuda`` takes. A row to ignore has loss and lse 0
    and is not read. A target outside the vocabulary gives NaN.

    Logits whose rows no single stride spans (logits[:, :-1] of a batch) are copied first: to leave a
    position out, give it the target ignore_index."""
    return _cross_entropy(logits, targets, int(ignore_index), float(label_smoothing), reduction, 1.0, want_lse=True)[:2]


def cross_entropy_with_grad_cuda(logits: Tensor, targets: Tensor, ignore_index: int = -100, label_smoothing: float = 0.0,
                                 reduction: str = "mean", grad_scale: float = 1.0, in_place: bool = False):
    """The loss ("mean" or "sum") and, in the same pass over the logits, their gradient.

    Returns (loss, grad): grad = grad_scale * d loss / d logits in logits' dtype (grad_scale: a loss
    scaler's factor), for ``logits.backward(grad)`` or a head's own backward; its rows are spaced as
    theirs where the padding is up to an eighth of a row. in_place writes it over the logits, which must
    then have rows that are contiguous inside, equally spaced and apart."""
    if reduction == "none":
        raise ValueError("a gradient needs a reduced loss (mean or sum)")
    _check_input("logits", logits)
    if in_place:
        if logits.dim() == 0:
            raise ValueError("logits must have a last dim (the vocabulary) that is not empty")
        if torch.is_grad_enabled() and logits.requires_grad:
            raise RuntimeError("in_place needs detached logits: autograd keeps their values")
        lr, stride = _rows(logits)
        if lr.data_ptr() != logits.data_ptr() or (logits.numel() > logits.shape[-1] and stride < logits.shape[-1]):
            raise ValueError("in_place needs logits whose rows are contiguous inside, equally spaced and apart")
        loss, _, _ = _cross_entropy(lr, targets, int(ignore_index), float(label_smoothing), reduction, float(grad_scale),
                                    in_place=True)
        _written([logits])
        return loss, logits
    loss, _, grad = _cross_entropy(logits, targets, int(ignore_index), float(label_smoothing), reduction, float(grad_scale),
                                   want_grad=True)
    return loss, grad


def cross_entropy_backward_cuda(grad_loss: Tensor, logits: Tensor, targets: Tensor, lse: Tensor, ignore_index: int = -100,
                                label_smoothing: float = 0.0, reduction: str = "mean"):
    """Gradient of ``cross_entropy_forward_cuda`` with respect to the logits, in their dtype,
    from the lse that it returned and the loss's gradient (a scalar, or of targets' shape for
    reduction "none"). One f32 lse leaves the softmax off by a factor of exp(half a unit in its
    last place), 2^-11 for logits of the order of 1e4; the other forms do not go through it."""
    return _cross_entropy_backward(grad_loss, logits, targets, lse, int(ignore_index), float(label_smoothing), reduction)


def _cross_entropy_backward(grad_loss, logits, targets, lse, ignore_index, label_smoothing, reduction, split=False):
    """split: lse is what ``_cross_entropy_split`` returned."""
    code, targets, kind, lr, stride = _loss_inputs(logits, targets, reduction)
    for name, t in (("lse", lse), ("grad_loss", grad_loss)):
        if not isinstance(t, Tensor) or t.device != logits.device:
            raise RuntimeError(f"{name} must be a tensor on {logits.device}")
    if not split and (lse.dtype != torch.float32 or lse.shape != targets.shape):
        raise ValueError(f"lse must be f32 of shape {tuple(targets.shape)}")
    if grad_loss.shape != targets.shape if kind == _lib.JK_REDUCE_NONE else grad_loss.numel() != 1:
        raise ValueError(f"grad_loss has shape {tuple(grad_loss.shape)}, which does not fit reduction {reduction!r}")
    gl = grad_loss.detach().to(torch.float32).contiguous()
    lse = lse.contiguous()
    grad = _grad_like(logits, lr, stride)
    work = _empty((_LIBRARY.jk_cross_entropy_workspace(targets.numel()) // 4,), torch.float32, logits.device)
    _call(_LIBRARY.jk_cross_entropy_backward_split, "jk_cross_entropy_backward_split", logits.get_device(), gl.data_ptr(),
          lr.data_ptr(), stride, targets.data_ptr(), lse.data_ptr(), lse.data_ptr() + 4 * targets.numel() if split else None,
          targets.numel(), logits.shape[-1], code, ignore_index, label_smoothing, kind, grad.data_ptr(), _rows(grad)[1], work.data_ptr())
    return grad


class _CrossEntropy(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, targets, ignore_index, label_smoothing, reduction):
        loss, lse = _cross_entropy_split(logits, targets, ignore_index, label_smoothing, reduction)
        ctx.save_for_backward(logits, targets, lse)
        ctx.options = (ignore_index, label_smoothing, reduction)
        return loss

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_loss):
        logits, targets, lse = ctx.saved_tensors
        return _cross_entropy_backward(grad_loss, logits, targets, lse, *ctx.options, split=True), None, None, None, None


def cross_entropy(logits: Tensor, targets: Tensor, ignore_index: int = -100, label_smoothing: float = 0.0,
                  reduction: str = "mean") -> Tensor:
    """Differentiable softmax cross entropy (f32): the loss of ``cross_entropy_forward_cuda`` and, in
    the backward pass, the gradient from the log-sum, which is kept in two f32. A loop that owns its
    backward pass reads the logits once less with ``cross_entropy_with_grad_cuda``."""
    return _CrossEntropy.apply(logits, targets, int(ignore_index), float(label_smoothing), reduction)


# ----------------------------------------------------------------------------- gradient norm
_NORM = {2.0: _lib.JK_NORM_2, math.inf: _lib.JK_NORM_INF}
_requires_grad = operator.attrgetter("requires_grad")
_CLIP_WORKSPACE = int(_LIBRARY.jk_clip_grad_norm_workspace()) // 8  # f64 elements


def _flat(t: Tensor) -> bool:
    """Whether t's elements fill one block of memory, in whatever order of its dims."""
    expected = 1
    for size, stride in sorted(((n, s) for n, s in zip(t.shape, t.stride()) if n != 1), key=lambda p: p[1]):
        if stride != expected:
            return False
        expected *= size
    return True


def _gradients(grads, name: str, only_gradients: bool = False) -> tuple[list[Tensor], list[torch.dtype]]:
    """The tensors, which are CUDA float tensors of one device, and their dtypes. only_gradients:
    parameters, and other leaves that autograd would refuse to change, are refused; a model's
    parameters, given in their gradients' place, would be scaled."""
    tensors = [grads] if isinstance(grads, Tensor) else list(grads)
    kinds = set(map(type, tensors))
    if type(None) in kinds:
        tensors = [g for g in tensors if g is not None]
        kinds.remove(type(None))
    if only_gradients and (kinds != {Tensor} or any(map(_requires_grad, tensors))):
        if any(isinstance(t, torch.nn.Parameter) or (isinstance(t, Tensor) and t.requires_grad and t.is_leaf) for t in tensors):
            raise TypeError("clip_grad_norm_ takes gradients, not parameters: [p.grad for p in parameters]")
    # one look at all of them (a model has hundreds); which one is wrong is sought only if one is
    try:
        devices = set(map(Tensor.get_device, tensors))  # -1: not a CUDA tensor
        types = [t.dtype for t in tensors]
        fine = len(devices) <= 1 and -1 not in devices and set(types) <= _DTYPE_CODE.keys()
    except TypeError:  # not a tensor
        fine = False
    if not fine:
        for i, t in enumerate(tensors):
            _check_input(f"{name} {i}", t)
            if t.device != tensors[0].device:
                raise RuntimeError(f"{name} {i} is on {t.device}, expected {tensors[0].device}")
    return tensors, types


def _codes(types: list[torch.dtype]) -> array.array:
    if types and types.count(types[0]) == len(types):
        return array.array("i", [_DTYPE_CODE[types[0]]]) * len(types)
    return array.array("i", map(_DTYPE_CODE.__getitem__, types))


def _addresses(tensors: list[Tensor]) -> array.array:
    return array.array("Q", map(Tensor.data_ptr, tensors))


def _refuse_twice(addresses: array.array, tensors: list[Tensor]) -> None:
    if len(set(addresses)) != len(addresses):  # empty tensors may share an address
        some = [p for p, t in zip(addresses, tensors) if t.numel()]
        if len(set(some)) != len(some):
            raise ValueError("a tensor is given twice: it would be scaled twice")


def _run_clip(tensors, types, outs, out_types, norm_type, clip, max_norm):
    kind = _NORM.get(float(norm_type))
    if kind is None:
        raise ValueError(f"unsupported norm_type {norm_type} (2 or inf)")
    src, dst, back = tensors, outs, None
    if not (all(map(Tensor.is_contiguous, tensors)) and (outs is None or all(map(Tensor.is_contiguous, outs)))):
        if clip:
            written = tensors if outs is None else outs
            for t in written:
                if any(s == 0 and n > 1 for n, s in zip(t.shape, t.stride())):
                    raise ValueError("a tensor to write has elements that share memory (an expanded tensor)")
            _refuse_twice(_addresses(written), written)
        src, dst, back = _blocks(tensors, outs, clip)
    ptrs, codes = _addresses(src), _codes(types)
    numels = array.array("q", map(Tensor.numel, src))
    out_ptrs, out_codes = (None, None) if dst is None else (_addresses(dst), _codes(out_types))
    if clip and back is None:
        _refuse_twice(ptrs if dst is None else out_ptrs, tensors)
    where = tensors[0].device if tensors else torch.device("cuda", _current_device())
    device = where.index
    work = _empty((_CLIP_WORKSPACE,), torch.float64, where)
    total = _empty((), torch.float32, where)
    _call(_LIBRARY.jk_clip_grad_norm, "jk_clip_grad_norm", device, ptrs.buffer_info()[0],
          None if dst is None else out_ptrs.buffer_info()[0], numels.buffer_info()[0], codes.buffer_info()[0],
          None if dst is None else out_codes.buffer_info()[0], len(src), kind, clip, max_norm, 1e-6, total.data_ptr(),
          work.data_ptr())
    if back:
        with torch.no_grad():
            for to, made in back:
                to.copy_(made)
    if clip:
        _written(tensors if outs is None else outs)
    return total


def _blocks(tensors, outs, clip):
    """(gradients, outs, copies to make after): a tensor that does not fill one block of memory is
    worked on in a contiguous copy, and an out whose elements lie in another order than its
    gradient's is written through one."""
    src, back = list(tensors), []
    dst = None if outs is None else list(outs)
    for i, g in enumerate(src):
        flat = _flat(g)
        if dst is None:
            if not flat:
                src[i] = g.detach().contiguous()
                if clip:
                    back.append((g, src[i]))
        elif not flat or dst[i].stride() != g.stride():
            src[i] = g.detach().contiguous()
            if not dst[i].is_contiguous():
                back.append((dst[i], torch.empty(g.shape, dtype=dst[i].dtype, device=g.device)))
                dst[i] = back[-1][1]
    return src, dst, back


def grad_norm(grads: Union[Tensor, Iterable[Optional[Tensor]]], norm_type: float = 2.0) -> Tensor:
    """Norm (2 or inf) over all elements of the gradients together, an f32 scalar on their
    device. Squares are added in f32 by up to 32 (in f64 where that would leave f32's range) and their
    sums in f64, so the norm is good to a few units of f32 and finite wherever it fits f32."""
    return _run_clip(*_gradients(grads, "gradient"), None, None, norm_type, 0, 0.0)


def clip_grad_norm_(grads: Union[Tensor, Iterable[Optional[Tensor]]], max_norm: float, norm_type: float = 2.0,
                    out: Optional[Iterable[Tensor]] = None, error_if_nonfinite: bool = False) -> Tensor:
    """Scales the gradients by ``min(1, max_norm / (norm + 1e-6))`` and returns the norm that
    they had (f32 scalar on their device, as ``grad_norm``).

    grads: one gradient or several (None is skipped; parameters are refused: they would be scaled
    themselves), in f32, bf16, f16 or a mix; scaled in place, or into `out`, one tensor for each gradient, of its shape and any of the three dtypes (f32
    master gradients of bf16 ones, say). Tensors must not overlap. A gradient that holds NaN
    makes all of them NaN, one that holds an infinity makes the others 0, as the formula has it;
    error_if_nonfinite raises instead, after reading the norm back, with the gradients scaled."""
    tensors, types = _gradients(grads, "gradient", only_gradients=True)
    outs = out_types = None
    if out is not None:
        outs, out_types = _gradients(out, "out", only_gradients=True)
        if len(outs) != len(tensors):
            raise ValueError(f"out has {len(outs)} tensors for {len(tensors)} gradients")
        if outs and outs[0].device != tensors[0].device:
            raise RuntimeError(f"out is on {outs[0].device}, expected {tensors[0].device}")
        if not all(map(Tensor.is_same_size, outs, tensors)):
            i = next(i for i, (o, g) in enumerate(zip(outs, tensors)) if o.shape != g.shape)
            raise ValueError(f"out {i} has shape {tuple(outs[i].shape)}, expected {tuple(tensors[i].shape)}")
    total = _run_clip(tensors, types, outs, out_types, norm_type, 1, float(max_norm))
    if error_if_nonfinite and not math.isfinite(total.item()):
        raise RuntimeError(f"the norm of the gradients is {total.item()}")
    return total
