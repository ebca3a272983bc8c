"""Dense operators on device arrays: layer norm, matrix products with an epilogue, log probabilities of
given tokens, each with its gradient.

They are what a model on top of the embeddings learns and answers with, beside the row normalisation
(``normalize_synapses``), the sparse window products and the ``softmax`` of the reference
(flyvec/core.py:17-36).  Arrays are :class:`flyvec_b200.engine.DeviceArray` or CUDA tensors of PyTorch; the
package itself does not import PyTorch.  Results are fresh dense arrays of the same kind.  Work is
enqueued on the current stream of the tensors' device (the default stream for ``DeviceArray``) and the calls
return at once; they may be captured into a CUDA graph.

Nothing here records a graph for automatic differentiation: tensors that require a gradient are refused
while gradients are enabled, and tensors with a forward-mode tangent always (pass ``x.detach()``).  The ``*_backward``
functions are called by hand or from a ``torch.autograd.Function``.

The last axis of every array is contiguous (``linear`` also takes a transposed ``x`` or ``weight``); leading axes
are taken together as rows and must lie at one common distance from one another.
"""
from __future__ import annotations

import ctypes as C
import sys
from functools import lru_cache
from typing import Any, NamedTuple

from . import _lib
from ._lib import ACTIVATIONS, DTYPES, check
from .engine import DeviceArray

__all__ = ["layer_norm", "layer_norm_backward", "linear", "linear_backward", "token_log_probs", "token_log_probs_backward",
           "TokenLogProbs", "MAX_TOP", "device_status"]

#: largest number of alternatives ``token_log_probs`` returns
MAX_TOP = 64

_FLOAT_MAX = (2 - 2.0 ** -23) * 2.0 ** 127
#: a beta has to be a positive float32 whose product with log2(e) is one too
_BETAS = 2.0 ** -149, 2.0 ** 127

_names: dict = {}  # dtype object -> name
_torch_types: dict = {}  # name -> torch dtype
_raw_stream = None  # (device) -> handle of the current stream
_forward_ad = None  # torch.autograd.forward_ad


def _type(x) -> str:
    name = _names.get(x.dtype)
    if name is None:
        name = _names[x.dtype] = str(x.dtype).replace("torch.", "")
    return name


def _has_tangent(x) -> bool:
    """Whether a tensor is one of forward-mode differentiation.  Outside of a level of it there are none: the question is
    asked of every argument, so that is looked at first (0.1 instead of 0.7 us)."""
    global _forward_ad
    if _forward_ad is None:
        _forward_ad = sys.modules["torch"].autograd.forward_ad
    return getattr(_forward_ad, "_current_level", 0) >= 0 and _forward_ad.unpack_dual(x).tangent is not None


def _refuse(x, what: str, types, like):
    """The error of an argument that :func:`_check` did not pass."""
    if not isinstance(x, DeviceArray):
        if not (hasattr(x, "data_ptr") and hasattr(x, "is_cuda") and hasattr(x, "is_neg")):
            raise TypeError(f"{what} must be a DeviceArray or a CUDA tensor, got {type(x).__name__}")
        if not x.is_cuda:
            raise ValueError(f"{what} must be on a GPU, got a tensor on {x.device}")
        if x.requires_grad and sys.modules["torch"].is_grad_enabled():
            raise ValueError(f"{what} requires a gradient, which these operators do not record: pass {what}.detach()")
        if _has_tangent(x):
            raise ValueError(f"{what} has a forward-mode tangent, which these operators do not carry on: pass {what}.detach()")
        if x.is_neg():
            raise ValueError(f"{what} is a lazily negated view: pass {what}.resolve_neg()")
    if _type(x) not in types:
        raise TypeError(f"{what} must have one of the types {', '.join(types)}, got {_type(x)}")
    if like is not None:
        if isinstance(x, DeviceArray) != isinstance(like, DeviceArray):
            raise TypeError(f"{what} is a {type(x).__name__}, the first argument a {type(like).__name__}")
        if x.get_device() != like.get_device():
            raise ValueError(f"{what} is on device {x.get_device()}, the first argument on device {like.get_device()}")


def _check(x, what: str, types, like=None):
    """One argument: a device array, of one of ``types``, on the device and of the kind of ``like``."""
    try:
        if x.is_cuda and not x.requires_grad and not x.is_neg() and _names.get(x.dtype) in types and (
                like is None or (type(x) is type(like) and x.get_device() == like.get_device())) and (
                isinstance(x, DeviceArray) or not _has_tangent(x)):
            return
    except AttributeError:
        pass
    _refuse(x, what, types, like)


def _rows(x, what: str):
    """(rows, columns, row stride) of an array whose leading axes are taken together."""
    shape, strides = x.shape, x.stride()
    if len(shape) == 2 and strides[1] == 1:
        return shape[0], shape[1], strides[0] if shape[0] != 1 else shape[1]
    if not len(shape):
        raise ValueError(f"{what} must have at least one axis")
    cols = shape[-1]
    if cols > 1 and strides[-1] != 1:
        raise ValueError(f"the last axis of {what} must be contiguous, its stride is {strides[-1]}: pass {what}.contiguous()")
    rows, step = 1, None
    for n, s in zip(reversed(shape[:-1]), reversed(strides[:-1])):
        if n != 1:
            if step is None:
                step = s
            elif s != step * rows and rows:
                raise ValueError(f"the leading axes of {what} (shape {tuple(shape)}, strides {strides}) do not lie at one common distance: "
                                 f"pass {what}.contiguous()")
        rows *= n
    return rows, cols, cols if step is None else step


def _matrix(x, what: str):
    """(rows, columns, row stride, column stride); two axes may be stored either way round."""
    shape = x.shape
    if len(shape) == 2:
        n, k = shape
        rs, cs = x.stride()
        if cs == 1 or k <= 1 or rs == 1 or n <= 1:
            return n, k, rs, cs
        raise ValueError(f"one axis of {what} must be contiguous, its strides are {(rs, cs)}: pass {what}.contiguous()")
    rows, cols, step = _rows(x, what)
    return rows, cols, step, 1


def _empty(like, shape, dtype: str):
    if isinstance(like, DeviceArray):
        return like.new_empty(shape, dtype)
    t = _torch_types.get(dtype)
    if t is None:
        t = _torch_types[dtype] = getattr(sys.modules["torch"], dtype)
    return like.new_empty(shape, dtype=t)


def _like(x):
    """A dense array of x's shape and type."""
    if not isinstance(x, DeviceArray) and x.is_contiguous():
        return sys.modules["torch"].empty_like(x)
    return _empty(x, x.shape, _type(x))


def _floats(like, n: int, shape):
    """n float32 arrays of one shape."""
    if isinstance(like, DeviceArray):
        return [like.new_empty(shape, "float32") for _ in range(n)]
    return _empty(like, (n, *shape), "float32").unbind(0)  # one allocation


def _stream(x, device: int):
    """Handle of the stream the work goes to."""
    global _raw_stream
    if isinstance(x, DeviceArray):
        return None
    if _raw_stream is None:
        torch = sys.modules["torch"]
        _raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda d: torch.cuda.current_stream(d).cuda_stream)
    return _raw_stream(device)


def _ptr(x):
    return None if x is None else x.data_ptr()


def _vector(x, n: int, what: str, like, types):
    """A dense vector of n elements (any shape of n elements is taken in order)."""
    _check(x, what, types, like)
    if x.numel() != n:
        raise ValueError(f"{what} must have {n} elements, got shape {tuple(x.shape)}")
    return x if x.is_contiguous() else x.contiguous()


def _row_vector(x, lead, rows: int, what: str, like, types):
    """A dense vector with one element a row, of the rows' own shape or on one axis: of [T, B] for rows [B, T] every element
    would go to another row."""
    x = _vector(x, rows, what, like, types)
    if len(x.shape) != 1:
        _same_shape(x, lead, what)
    return x


def _same_shape(x, shape, what: str):
    if tuple(x.shape) != tuple(shape):
        raise ValueError(f"{what} must have shape {tuple(shape)}, got {tuple(x.shape)}")


def _activation(name) -> int:
    code = ACTIVATIONS.get("none" if name is None else name)
    if code is None:
        raise ValueError(f"activation must be one of {', '.join(ACTIVATIONS)}, got {name!r}")
    return code


# workspace sizes: functions of sizes, strides and the alignment of the operands alone
@lru_cache(maxsize=1024)
def _norm_workspace(device: int, rows: int, cols: int, dtype: int) -> int:
    need = C.c_size_t(0)
    check(_lib.lib().fv_layer_norm_backward_workspace(device, rows, cols, dtype, C.byref(need)))
    return need.value


@lru_cache(maxsize=1024)
def _linear_workspace(rows: int, inner: int, outer: int, x: int, xr: int, xc: int, w: int, wr: int, wc: int) -> int:
    need = C.c_size_t(0)
    check(_lib.lib().fv_linear_workspace(rows, inner, outer, x, xr, xc, w, wr, wc, C.byref(need)))
    return need.value


@lru_cache(maxsize=1024)
def _linear_backward_workspace(device: int, rows: int, inner: int, outer: int, dy: int, gs: int, x: int, xr: int, xc: int, w: int, wr: int,
                               wc: int, act: int) -> int:
    need = C.c_size_t(0)
    check(_lib.lib().fv_linear_backward_workspace(device, rows, inner, outer, dy, gs, x, xr, xc, w, wr, wc, act, C.byref(need)))
    return need.value


# ---- layer norm ------------------------------------------------------------------------------------
def layer_norm(x, weight=None, bias=None, eps: float = 1e-5, out_dtype: str | None = None, return_stats: bool = False):
    """``(x - mean) / sqrt(var + eps) * weight + bias`` over the last axis.

    ``x``: float32, bfloat16 or float16; ``weight`` and ``bias`` of the same type (a bias needs a weight).  The result
    has ``x``'s type or ``out_dtype``.  With ``return_stats`` the float32 mean and ``1 / sqrt(var + eps)`` of every row
    come back too, for :func:`layer_norm_backward`."""
    _check(x, "x", DTYPES)
    rows, cols, step = _rows(x, "x")
    kind = _type(x)
    out_dtype = kind if out_dtype is None else out_dtype
    if out_dtype not in DTYPES:
        raise TypeError(f"out_dtype must be one of {', '.join(DTYPES)}, got {out_dtype!r}")
    if cols == 0:
        raise ValueError("x has no columns")
    if not 0 <= eps <= _FLOAT_MAX:
        raise ValueError(f"eps must be a finite float32 and not negative, got {eps}")
    if bias is not None and weight is None:
        raise ValueError("a bias needs a weight")
    if weight is not None:
        weight = _vector(weight, cols, "weight", x, (kind,))
    if bias is not None:
        bias = _vector(bias, cols, "bias", x, (kind,))
    y, mean, rstd, dev = _like(x) if out_dtype == kind else _empty(x, x.shape, out_dtype), None, None, x.get_device()
    if return_stats:
        lead = x.shape[:-1]
        mean, rstd = _empty(x, lead, "float32"), _empty(x, lead, "float32")
    check(_lib.lib().fv_layer_norm(dev, _stream(x, dev), x.data_ptr(), step, rows, cols, DTYPES[kind], _ptr(weight), _ptr(bias), eps,
                                   y.data_ptr(), DTYPES[out_dtype], _ptr(mean), _ptr(rstd)))
    return (y, mean, rstd) if return_stats else y


def layer_norm_backward(dy, x, mean, rstd, weight=None):
    """``(dx, dweight, dbias)`` of :func:`layer_norm` from the gradient ``dy`` of its result and the statistics it
    returned (shaped like ``x`` without its last axis, or flat); without a weight the last two are None.  The weight's
    gradients are sums over all rows, formed in float32 in a fixed order and rounded once."""
    _check(x, "x", DTYPES)
    rows, cols, step = _rows(x, "x")
    kind = _type(x)
    if cols == 0:
        raise ValueError("x has no columns")
    _check(dy, "dy", (kind,), x)
    _same_shape(dy, x.shape, "dy")
    _, _, gstep = _rows(dy, "dy")
    mean = _row_vector(mean, x.shape[:-1], rows, "mean", x, ("float32",))
    rstd = _row_vector(rstd, x.shape[:-1], rows, "rstd", x, ("float32",))
    if weight is not None:
        weight = _vector(weight, cols, "weight", x, (kind,))
    dx = _like(x)
    dev, lib = x.get_device(), _lib.lib()
    dw = db = ws = None
    size = 0
    if weight is not None:
        size = _norm_workspace(dev, rows, cols, DTYPES[kind])
        dw, db, ws = _empty(x, (cols,), kind), _empty(x, (cols,), kind), _empty(x, (size,), "uint8")
    check(lib.fv_layer_norm_backward(dev, _stream(x, dev), dy.data_ptr(), gstep, x.data_ptr(), step, rows, cols, DTYPES[kind], mean.data_ptr(),
                                     rstd.data_ptr(), _ptr(weight), dx.data_ptr(), _ptr(dw), _ptr(db), _ptr(ws), size))
    return dx, dw, db


# ---- matrix product --------------------------------------------------------------------------------
_HALF = ("bfloat16", "float16")


def linear(x, weight, bias=None, activation: str | None = None, residual=None, out_dtype: str | None = None,
           return_preactivation: bool = False):
    """``act(x @ weight.T + bias) + residual``.

    ``x`` ``[..., inner]`` and ``weight`` ``[outer, inner]`` are bfloat16 or float16, ``bias`` ``[outer]`` and ``residual``
    ``[..., outer]`` of the same type; ``activation`` is "none", "relu", "gelu", "gelu_tanh" or "silu".  Products are summed in
    float32; the result is rounded once to the operands' type, or comes as ``out_dtype="float32"``.  With
    ``return_preactivation`` the value before the activation comes back too, for :func:`linear_backward`."""
    _check(x, "x", _HALF)
    kind = _type(x)
    _check(weight, "weight", (kind,), x)
    if len(weight.shape) != 2:
        raise ValueError(f"weight must have shape [outer, inner], got {tuple(weight.shape)}")
    rows, inner, xr, xc = _matrix(x, "x")
    outer, winner, wr, wc = _matrix(weight, "weight")
    if winner != inner:
        raise ValueError(f"x has {inner} columns, the weight {winner}")
    if inner == 0 or outer == 0:
        raise ValueError("x and the weight must not be empty")
    act = _activation(activation)
    out_dtype = kind if out_dtype is None else out_dtype
    if out_dtype not in (kind, "float32"):
        raise TypeError(f"out_dtype must be {kind} or float32, got {out_dtype!r}")
    if bias is not None:
        bias = _vector(bias, outer, "bias", x, (kind,))
    shape = tuple(x.shape[:-1]) + (outer,)
    rstep = 0
    if residual is not None:
        _check(residual, "residual", (kind,), x)
        _same_shape(residual, shape, "residual")
        _, _, rstep = _rows(residual, "residual")
    y = _empty(x, shape, out_dtype)
    z = _empty(x, shape, kind) if return_preactivation else None
    dev, px, pw = x.get_device(), x.data_ptr(), weight.data_ptr()
    size = _linear_workspace(rows, inner, outer, px & 15, xr, xc, pw & 15, wr, wc)
    ws = _empty(x, (size,), "uint8") if size else None
    check(_lib.lib().fv_linear(dev, _stream(x, dev), px, xr, xc, pw, wr, wc, rows, inner, outer, DTYPES[kind], _ptr(bias), act,
                               _ptr(residual), rstep, y.data_ptr(), DTYPES[out_dtype], _ptr(z), _ptr(ws), size))
    return (y, z) if return_preactivation else y


def linear_backward(dy, x, weight, preactivation=None, activation: str | None = None):
    """``(dx, dweight, dbias)`` of :func:`linear` from the gradient ``dy`` of its result.  With an activation the
    pre-activation that the forward call returned is needed.  The residual's gradient is ``dy`` itself."""
    _check(x, "x", _HALF)
    kind = _type(x)
    _check(weight, "weight", (kind,), x)
    if len(weight.shape) != 2:
        raise ValueError(f"weight must have shape [outer, inner], got {tuple(weight.shape)}")
    rows, inner, xr, xc = _matrix(x, "x")
    outer, winner, wr, wc = _matrix(weight, "weight")
    if winner != inner:
        raise ValueError(f"x has {inner} columns, the weight {winner}")
    if inner == 0 or outer == 0:
        raise ValueError("x and the weight must not be empty")
    act = _activation(activation)
    shape = tuple(x.shape[:-1]) + (outer,)
    _check(dy, "dy", (kind,), x)
    _same_shape(dy, shape, "dy")
    _, _, gstep = _rows(dy, "dy")
    zstep = 0
    if act:
        if preactivation is None:
            raise ValueError(f"the gradient of {activation} needs the pre-activation")
        _check(preactivation, "preactivation", (kind,), x)
        _same_shape(preactivation, shape, "preactivation")
        _, _, zstep = _rows(preactivation, "preactivation")
    else:
        preactivation = None
    dx, dw, db = _like(x), _empty(x, (outer, inner), kind), _empty(x, (outer,), kind)
    dev, pg, px, pw = x.get_device(), dy.data_ptr(), x.data_ptr(), weight.data_ptr()
    size = _linear_backward_workspace(dev, rows, inner, outer, pg & 15, gstep, px & 15, xr, xc, pw & 15, wr, wc, act)
    ws = _empty(x, (size,), "uint8") if size else None
    check(_lib.lib().fv_linear_backward(dev, _stream(x, dev), pg, gstep, px, xr, xc, pw, wr, wc, rows, inner, outer, DTYPES[kind],
                                        _ptr(preactivation), zstep, act, dx.data_ptr(), dw.data_ptr(), db.data_ptr(), _ptr(ws), size))
    return dx, dw, db


# ---- log probabilities -----------------------------------------------------------------------------
_INTS = ("int32", "int64")


class TokenLogProbs(NamedTuple):
    """What :func:`token_log_probs` answers, float32 except the int32 ``top_ids``; the last two are None for ``top=0``."""
    log_prob: Any
    entropy: Any
    row_max: Any
    log_z: Any
    top_ids: Any
    top_log_prob: Any


def token_log_probs(logits, targets, beta: float = 1.0, top: int = 0) -> TokenLogProbs:
    """Log probability of one given token per row under ``softmax(beta * logits)``, with the row's entropy and its ``top``
    most probable tokens (larger logit first, ties to the lower id) with their log probabilities.

    ``logits`` ``[..., vocab]`` float32, bfloat16 or float16; ``targets`` ``[...]`` int32 or int64, -1 for padding (log
    probability 0), NaN for any other id outside the vocabulary.  ``row_max`` and ``log_z`` (the log of the sum of
    ``exp(beta * (logits - row_max))``) go to :func:`token_log_probs_backward`.  A row of -inf only has log
    probabilities -inf, entropy 0 and ``log_z`` -inf; a row with a NaN or +inf has NaN everywhere but in ``top_ids``, which
    take NaN as the largest."""
    _check(logits, "logits", DTYPES)
    rows, vocab, step = _rows(logits, "logits")
    if vocab == 0:
        raise ValueError("the vocabulary is empty")
    if not _BETAS[0] <= beta <= _BETAS[1]:
        raise ValueError(f"beta must be between 2^-149 and 2^127, got {beta}")
    if not 0 <= top <= min(MAX_TOP, vocab):
        raise ValueError(f"top must be between 0 and min({MAX_TOP}, {vocab}), got {top}")
    lead = tuple(logits.shape[:-1])
    targets = _vector(targets, rows, "targets", logits, _INTS)
    _same_shape(targets, lead, "targets")
    lp, ent, mx, lz = _floats(logits, 4, lead)
    dev = logits.get_device()
    ids = _empty(logits, lead + (top,), "int32") if top else None
    tlp = _empty(logits, lead + (top,), "float32") if top else None
    check(_lib.lib().fv_token_log_probs(dev, _stream(logits, dev), logits.data_ptr(), step, rows, vocab, DTYPES[_type(logits)],
                                        targets.data_ptr(), int(_type(targets) == "int64"), beta, top, lp.data_ptr(), ent.data_ptr(),
                                        mx.data_ptr(), lz.data_ptr(), _ptr(ids), _ptr(tlp)))
    return TokenLogProbs(lp, ent, mx, lz, ids, tlp)


def token_log_probs_backward(grad_log_prob, logits, targets, row_max, log_z, entropy=None, grad_entropy=None, beta: float = 1.0):
    """Gradient by the logits (in their type) of ``sum(grad_log_prob * log_prob) + sum(grad_entropy * entropy)``; ``row_max``,
    ``log_z`` and, where the entropy has a gradient, ``entropy`` as :func:`token_log_probs` returned them, and the gradients, are
    float32 and shaped like ``targets`` or flat.  Padding
    rows get the entropy's part only, rows of -inf only get zeros."""
    _check(logits, "logits", DTYPES)
    rows, vocab, step = _rows(logits, "logits")
    if vocab == 0:
        raise ValueError("the vocabulary is empty")
    if not _BETAS[0] <= beta <= _BETAS[1]:
        raise ValueError(f"beta must be between 2^-149 and 2^127, got {beta}")
    lead, f32 = logits.shape[:-1], ("float32",)
    targets = _vector(targets, rows, "targets", logits, _INTS)
    _same_shape(targets, lead, "targets")
    grad_log_prob = _row_vector(grad_log_prob, lead, rows, "grad_log_prob", logits, f32)
    row_max, log_z = _row_vector(row_max, lead, rows, "row_max", logits, f32), _row_vector(log_z, lead, rows, "log_z", logits, f32)
    if grad_entropy is not None:
        if entropy is None:
            raise ValueError("the entropy's gradient needs the entropy")
        grad_entropy = _row_vector(grad_entropy, lead, rows, "grad_entropy", logits, f32)
        entropy = _row_vector(entropy, lead, rows, "entropy", logits, f32)
    else:
        entropy = None
    dx, dev = _like(logits), logits.get_device()
    check(_lib.lib().fv_token_log_probs_backward(dev, _stream(logits, dev), grad_log_prob.data_ptr(), _ptr(grad_entropy),
                                                 logits.data_ptr(), step, rows, vocab, DTYPES[_type(logits)], targets.data_ptr(),
                                                 int(_type(targets) == "int64"), row_max.data_ptr(), log_z.data_ptr(), _ptr(entropy), beta,
                                                 dx.data_ptr()))
    return dx


def device_status(device: int = 0) -> int:
    """Error bits the operators' kernels raised on ``device`` since the last call (0: none; bit 0: a bounded wait
    inside a kernel ran out and its results are invalid).  Waits for the device and clears the bits."""
    word = C.c_uint32(0)
    check(_lib.lib().fv_ops_status(device, C.byref(word)))
    return word.value
