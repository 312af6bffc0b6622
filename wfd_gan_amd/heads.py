"""Tensor-level entry points of the classifier-head kernels (include/wfdgan.h, "classifier head"): layer norm with its
backward, the scores of given labels over many classes (log probability, entropy, top alternatives) with their gradient, and the
loss of a student that learns from a teacher's top logits.

Rows lie along the last dimension and may be float32, bfloat16 or float16; leading dimensions are free; rows with a stride are
read where they are, anything else is copied first.  As everywhere in this package the backward is a call of its own in closed
form (no autograd graph), there is no CPU path, and a call only enqueues work on the current stream of the tensors' device.

Results go into fresh tensors, or into those of an earlier call's result passed as ``out=`` (same sizes): then a call allocates
nothing, which is what a loop or a captured graph wants.  What such a call does not write (no ``stats``, no labels, ``k`` = 0, no
``grad``) is None in what it returns.  A result belongs to one call in flight: give calls that may overlap (other streams, graphs
that replay side by side) results of their own.
"""
from __future__ import annotations

from functools import lru_cache
from typing import NamedTuple, Optional

import torch

from ._lib import lib

MAX_ALTERNATIVES = 64
MAX_TEACHER_ENTRIES = 256
_CODES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_INT32 = 1 << 31


class NormOutput(NamedTuple):
    y: torch.Tensor
    mean: Optional[torch.Tensor]          # fp32, one per row: what the backward needs
    rstd: Optional[torch.Tensor]


class NormGradients(NamedTuple):
    dx: torch.Tensor
    dweight: Optional[torch.Tensor]
    dbias: Optional[torch.Tensor]
    work: torch.Tensor


class LabelScores(NamedTuple):
    logprob: Optional[torch.Tensor]       # fp32, shape of the labels
    entropy: Optional[torch.Tensor]
    stat: Optional[torch.Tensor]          # fp32 (..., 2): row maximum, log of the sum of exponentials about it
    top_logprob: Optional[torch.Tensor]   # fp32 (..., k)
    top_index: Optional[torch.Tensor]     # int32 (..., k)
    work: Optional[torch.Tensor]


class DistillOutput(NamedTuple):
    loss: torch.Tensor                    # fp32, one per row
    dlogits: Optional[torch.Tensor]
    work: Optional[torch.Tensor]


# ---- argument checks -------------------------------------------------------------------------------------------------
def _code(t: torch.Tensor, name: str) -> int:
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name}: expected a tensor, got {type(t).__name__}")
    c = _CODES.get(t.dtype)
    if c is None:
        raise TypeError(f"{name}: float32, bfloat16 or float16 rows, got {t.dtype}")
    return c


def _no_rows(t: torch.Tensor, name: str):
    if not t.shape or t.shape[-1] == 0:
        raise ValueError(f"{name}: needs a last dimension of at least one element, got shape {tuple(t.shape)}")
    raise ValueError(f"{name}: {t.numel() // t.shape[-1]} rows of {t.shape[-1]} are more than 2^31 - 1")


def _sizes(t: torch.Tensor, name: str):
    """(rows, columns) of rows whose buffers are asked for, checked as _rows does"""
    n = t.shape[-1] if t.shape else 0
    m = t.numel() // n if n else 0
    if n == 0 or m >= _INT32 or n >= _INT32:
        _no_rows(t, name)
    return m, n


def _rows(t: torch.Tensor, name: str):
    """(tensor whose storage is read, rows, columns, row stride)"""
    shape = t.shape
    if not shape or shape[-1] == 0:
        _no_rows(t, name)
    n = shape[-1]
    m = t.numel() // n
    if m >= _INT32 or n >= _INT32:
        _no_rows(t, name)
    if t.is_contiguous():
        return t, m, n, n
    if len(shape) == 2 and (t.stride(1) == 1 or n == 1) and n <= t.stride(0) < _INT32:
        return t, m, n, t.stride(0)
    return t.contiguous(), m, n, n


def _device(t: torch.Tensor, who: str, *others) -> int:
    """The GPU's index, the same for all operands."""
    i = t.get_device()
    for o in others:
        if o is not None and o.get_device() != i:
            raise ValueError(f"{who}: an operand of shape {tuple(o.shape)} is on {o.device}, the rows are on {t.device}")
    if i < 0:
        raise RuntimeError(f"{who}: these kernels run on the MI355X only (got a {t.device} tensor); there is no CPU fallback")
    return i


def _vector(t, who: str, name: str, numel: int, dtype) -> torch.Tensor:
    """An optional per-row or per-column operand: its dtype and size checked, contiguous."""
    if t is None:
        return None
    if not isinstance(t, torch.Tensor) or t.dtype != dtype:
        raise TypeError(f"{who}: {name} must be a {dtype} tensor, got {getattr(t, 'dtype', type(t).__name__)}")
    if t.numel() != numel:
        raise ValueError(f"{who}: {name} has {t.numel()} elements, expected {numel}")
    return t if t.is_contiguous() else t.contiguous()


def _wide(shape) -> list:
    return [n for n in shape if n != 1]


def _in_order(rows: torch.Tensor, who: str, **operands):
    """Rows with several leading dimensions: a per-row operand (``name_2``: of two elements each) has the same ones, or a single
    one, dimensions of 1 aside; any other shape of as many elements would be read in another order than it is meant."""
    lead = rows.shape[:-1]
    for name, t in operands.items():
        if t is None or t.dim() < 2:
            continue
        last = (2,) if name.endswith("_2") else ()
        if _wide(t.shape) not in (_wide((*lead, *last)), _wide((lead.numel(), *last))):
            raise ValueError(f"{who}: {name[:-2] if last else name} has shape {tuple(t.shape)}, the rows' is {tuple(lead)}")


def _result(t, who: str, name: str, numel: int, dtype, dev: int) -> int:
    """The address of one tensor of an earlier result that is written again."""
    if t is None or t.dtype != dtype or t.numel() != numel or t.get_device() != dev or not t.is_contiguous():
        got = None if t is None else (t.dtype, tuple(t.shape), t.device)
        raise ValueError(f"{who}: out.{name} must be a contiguous {dtype} tensor of {numel} elements on cuda:{dev}, got {got}")
    return t.data_ptr()


def _scratch(t, who: str, floats: int, dev: int) -> int:
    if floats == 0:
        return 0
    if t is None or t.dtype != torch.float32 or t.numel() < floats or t.get_device() != dev or not t.is_contiguous():
        raise ValueError(f"{who}: out.work must hold {floats} float32 on cuda:{dev} (take out from a call of these sizes)")
    return t.data_ptr()


@lru_cache(maxsize=1024)
def _floats(which: str, *sizes) -> int:
    """How much scratch a call of these sizes needs (a function of the sizes alone)."""
    return getattr(lib(), which)(*sizes)


def _ptr(t) -> int:
    return 0 if t is None else t.data_ptr()


# The current device and the current stream's handle without the objects around them: 0.1 us instead of 2.1 of a call that takes 6.
_current = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device
_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda i: torch.cuda.current_stream(i).cuda_stream)


def _launch(dev: int, fn, *args):
    if dev == _current():
        fn(*args, _stream(dev))
        return
    with torch.cuda.device(dev):
        fn(*args, _stream(dev))


def _temperature(t: float, who: str) -> float:
    t = float(t)
    if not 1e-6 <= t <= 1e6:
        raise ValueError(f"{who}: temperature must be in [1e-6, 1e6], got {t}")
    return t


# ---- layer norm --------------------------------------------------------------------------------------------------------
def _norm_weights(who, code, n, weight, bias):
    """(their dtype, weight, bias), both optional"""
    t = weight if weight is not None else bias
    if t is None:
        return torch.float32, None, None
    wd = getattr(t, "dtype", None)
    if wd != torch.float32 and _CODES.get(wd) != code:
        raise TypeError(f"{who}: weight and bias must be float32 or have the rows' dtype, got {wd}")
    if weight is not None and bias is not None and getattr(bias, "dtype", None) != wd:
        raise TypeError(f"{who}: weight and bias must have one dtype, got {wd} and {getattr(bias, 'dtype', type(bias).__name__)}")
    return wd, _vector(weight, who, "weight", n, wd), _vector(bias, who, "bias", n, wd)


def norm_output_like(x: torch.Tensor, stats: bool = True) -> NormOutput:
    """Buffers for ``layer_norm(x, ..., out=...)``."""
    _code(x, "x")
    _sizes(x, "x")
    lead = x.shape[:-1]
    f = dict(dtype=torch.float32, device=x.device)
    return NormOutput(torch.empty(x.shape, dtype=x.dtype, device=x.device), torch.empty(lead, **f) if stats else None,
                      torch.empty(lead, **f) if stats else None)


def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None, eps: float = 1e-5,
               *, stats: bool = True, out: Optional[NormOutput] = None) -> NormOutput:
    """``(x - mean) * rstd * weight + bias`` over the last dimension; mean and rstd are returned for the backward unless
    ``stats`` is false.  ``out.y`` may be ``x``."""
    who = "layer_norm"
    code = _code(x, "x")
    xr, m, n, ld = _rows(x, "x")
    wd, w, b = _norm_weights(who, code, n, weight, bias)
    eps = float(eps)
    if not eps >= 0.0:
        raise ValueError(f"{who}: eps must not be negative, got {eps}")
    dev = _device(x, who, w, b)
    if out is None:
        out = norm_output_like(x, stats)
    y = _result(out.y, who, "y", m * n, x.dtype, dev)
    mean = _result(out.mean, who, "mean", m, torch.float32, dev) if stats else 0
    rstd = _result(out.rstd, who, "rstd", m, torch.float32, dev) if stats else 0
    _launch(dev, lib().layer_norm_fwd, xr.data_ptr(), ld, code, _ptr(w), _ptr(b), _CODES[wd], m, n, eps, y, n, mean, rstd)
    return out if stats or out.mean is out.rstd is None else out._replace(mean=None, rstd=None)


def norm_gradients_like(x: torch.Tensor, weight: Optional[torch.Tensor] = None,
                        bias: Optional[torch.Tensor] = None) -> NormGradients:
    """Buffers for ``layer_norm_backward(..., out=...)``; without a weight (bias) there is no dweight (dbias)."""
    code = _code(x, "x")
    m, n = _sizes(x, "x")
    floats = _floats("layer_norm_bwd_floats", m, n, code)
    if floats < 0:
        raise ValueError(f"layer_norm_backward: rows of {n} are not supported")
    grad = lambda w: None if w is None else torch.empty(n, dtype=w.dtype, device=x.device)
    return NormGradients(torch.empty(x.shape, dtype=x.dtype, device=x.device), grad(weight), grad(bias),
                         torch.empty(floats, dtype=torch.float32, device=x.device))


def layer_norm_backward(dy: torch.Tensor, x: torch.Tensor, weight: Optional[torch.Tensor], mean: torch.Tensor,
                        rstd: torch.Tensor, *, bias: bool = True, out: Optional[NormGradients] = None) -> NormGradients:
    """Gradients of ``layer_norm`` from its saved mean and rstd: dx in the rows' dtype, dweight and dbias in the weight's (both
    float32 without a weight, where dweight is None); sums over the rows are fp32 in a fixed order.  ``out.dx`` may be ``dy`` or
    ``x``."""
    who = "layer_norm_backward"
    code = _code(x, "x")
    if _code(dy, "dy") != code or dy.shape != x.shape:
        raise ValueError(f"{who}: dy {dy.dtype} {tuple(dy.shape)} does not match x {x.dtype} {tuple(x.shape)}")
    xr, m, n, ldx = _rows(x, "x")
    dyr, _, _, lddy = _rows(dy, "dy")
    wd, w, _ = _norm_weights(who, code, n, weight, None)
    if mean is None or rstd is None:
        raise ValueError(f"{who}: needs the mean and rstd that layer_norm returned")
    mean, rstd = _vector(mean, who, "mean", m, torch.float32), _vector(rstd, who, "rstd", m, torch.float32)
    if x.dim() > 2:
        _in_order(x, who, mean=mean, rstd=rstd)
    dev = _device(x, who, dyr, w, mean, rstd)
    if out is None:
        like = torch.empty(0, dtype=wd, device=x.device)
        out = norm_gradients_like(x, w, like if bias else None)
    dx = _result(out.dx, who, "dx", m * n, x.dtype, dev)
    dw = 0 if out.dweight is None else _result(out.dweight, who, "dweight", n, wd, dev)
    db = 0 if out.dbias is None else _result(out.dbias, who, "dbias", n, wd, dev)
    work = _scratch(out.work, who, _floats("layer_norm_bwd_floats", m, n, code), dev)
    _launch(dev, lib().layer_norm_bwd, dyr.data_ptr(), lddy, xr.data_ptr(), ldx, code, _ptr(w), _CODES[wd], mean.data_ptr(),
            rstd.data_ptr(), m, n, dx, n, dw, db, work)
    return out


# ---- scores of given labels ------------------------------------------------------------------------------------------
def scores_like(logits: torch.Tensor, k: int = 0) -> LabelScores:
    """Buffers for ``label_logprobs(logits, ..., k, out=...)``."""
    code = _code(logits, "logits")
    m, v = _sizes(logits, "logits")
    floats = _floats("label_scores_floats", m, v, code, k) if 0 <= k <= MAX_ALTERNATIVES else -1
    if floats < 0:
        raise ValueError(f"label_logprobs: {k} alternatives of {v} classes are not supported (at most {MAX_ALTERNATIVES})")
    lead, dev = logits.shape[:-1], logits.device
    f = dict(dtype=torch.float32, device=dev)
    return LabelScores(torch.empty(lead, **f), torch.empty(lead, **f), torch.empty(*lead, 2, **f),
                       torch.empty(*lead, k, **f) if k else None,
                       torch.empty(*lead, k, dtype=torch.int32, device=dev) if k else None,
                       torch.empty(floats, **f) if floats else None)


def label_logprobs(logits: torch.Tensor, labels: Optional[torch.Tensor], k: int = 0, *, temperature: float = 1.0,
                   out: Optional[LabelScores] = None) -> LabelScores:
    """Log probability of each row's label under softmax(logits / temperature), the entropy of that distribution and its ``k``
    largest classes in order (equal logits: the lower index first), all in one pass over the logits.

    ``labels``: int32, one per row; negative = no label (log probability 0), >= classes = NaN; None: no ``logprob``.
    A row of nothing but -inf has log probabilities -inf and entropy 0; one with NaN or +inf is NaN."""
    who = "label_logprobs"
    code = _code(logits, "logits")
    xr, m, v, ld = _rows(logits, "logits")
    k = int(k)
    if not 0 <= k <= min(v, MAX_ALTERNATIVES):
        raise ValueError(f"{who}: k must be 0 .. {min(v, MAX_ALTERNATIVES)}, got {k}")
    y = _vector(labels, who, "labels", m, torch.int32)
    if logits.dim() > 2:
        _in_order(logits, who, labels=y)
    temperature = _temperature(temperature, who)
    dev = _device(logits, who, y)
    if out is None:
        out = scores_like(logits, k)
    f32 = torch.float32
    lp = 0 if y is None else _result(out.logprob, who, "logprob", m, f32, dev)
    ent = 0 if out.entropy is None else _result(out.entropy, who, "entropy", m, f32, dev)
    stat = 0 if out.stat is None else _result(out.stat, who, "stat", 2 * m, f32, dev)
    top = _result(out.top_logprob, who, "top_logprob", m * k, f32, dev) if k else 0
    idx = _result(out.top_index, who, "top_index", m * k, torch.int32, dev) if k else 0
    work = _scratch(out.work, who, _floats("label_scores_floats", m, v, code, k), dev)
    _launch(dev, lib().label_scores, xr.data_ptr(), ld, code, m, v, _ptr(y), temperature, k, lp, ent, stat, top, idx, work)
    if y is None and out.logprob is not None:
        out = out._replace(logprob=None)
    if k == 0 and (out.top_logprob is not None or out.top_index is not None):
        out = out._replace(top_logprob=None, top_index=None)
    return out


def label_logprobs_backward(logits: torch.Tensor, labels: Optional[torch.Tensor], scores: LabelScores,
                            d_logprob: Optional[torch.Tensor], d_entropy: Optional[torch.Tensor] = None, *,
                            temperature: float = 1.0, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Gradient of ``(d_logprob * logprob + d_entropy * entropy).sum()`` with respect to the logits.  ``scores`` is what
    ``label_logprobs`` returned for these logits at this temperature (its stat and, with ``d_entropy``, its entropy are read).
    ``out`` may be ``logits`` itself."""
    who = "label_logprobs_backward"
    code = _code(logits, "logits")
    xr, m, v, ld = _rows(logits, "logits")
    y = _vector(labels, who, "labels", m, torch.int32)
    if d_logprob is not None and y is None:
        raise ValueError(f"{who}: d_logprob needs the labels")
    if scores.stat is None or (d_entropy is not None and scores.entropy is None):
        raise ValueError(f"{who}: scores lacks the stat or entropy that label_logprobs returned")
    stat = _vector(scores.stat, who, "scores.stat", 2 * m, torch.float32)
    ent = _vector(scores.entropy, who, "scores.entropy", m, torch.float32) if d_entropy is not None else None
    dl, dh = _vector(d_logprob, who, "d_logprob", m, torch.float32), _vector(d_entropy, who, "d_entropy", m, torch.float32)
    if logits.dim() > 2:
        _in_order(logits, who, labels=y, stat_2=stat, entropy=ent, d_logprob=dl, d_entropy=dh)
    temperature = _temperature(temperature, who)
    dev = _device(logits, who, y, stat, ent, dl, dh)
    if out is None:
        out = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
    dx = _result(out, who, "dlogits", m * v, logits.dtype, dev)
    _launch(dev, lib().label_scores_bwd, xr.data_ptr(), ld, code, m, v, _ptr(y), temperature, stat.data_ptr(), _ptr(ent),
            _ptr(dl), _ptr(dh), dx, v)
    return out


# ---- distillation ------------------------------------------------------------------------------------------------------
def distill_output_like(logits: torch.Tensor, grad: bool = True) -> DistillOutput:
    """Buffers for ``distill_loss(logits, ..., out=...)``."""
    code = _code(logits, "logits")
    m, v = _sizes(logits, "logits")
    floats = _floats("distill_floats", m, v, code)
    if floats < 0:
        raise ValueError(f"distill_loss: {v} classes are not supported")
    f = dict(dtype=torch.float32, device=logits.device)
    return DistillOutput(torch.empty(logits.shape[:-1], **f),
                         torch.empty(logits.shape, dtype=logits.dtype, device=logits.device) if grad else None,
                         torch.empty(floats, **f) if floats else None)


def distill_loss(logits: torch.Tensor, teacher_index: torch.Tensor, teacher_value: torch.Tensor,
                 labels: Optional[torch.Tensor] = None, *, temperature: float = 1.0, weight: float = 1.0,
                 label_weight: float = 0.0, row_scale: Optional[torch.Tensor] = None, grad_scale: float = 1.0, grad: bool = True,
                 out: Optional[DistillOutput] = None) -> DistillOutput:
    """Per-row loss of a student against a teacher's top logits, and its gradient in the same call:

        weight * T^2 * KL(softmax(teacher_value / T) || softmax(logits / T) at teacher_index) - label_weight * ln softmax(logits)[label]

    ``teacher_index`` (int32) and ``teacher_value`` (float32: logits or log probabilities, their offset does not matter) are
    (..., K) with K <= 256; an index < 0 is no entry, an index that occurs twice counts twice.  ``labels`` (int32) are needed
    when ``label_weight`` is not 0; negative = no label.  A row with neither entry nor label has loss and gradient 0 whatever it
    holds.  ``dlogits`` carries ``grad_scale * row_scale`` (the losses do not).
    An index or label >= classes makes its row NaN.  ``out.dlogits`` may be ``logits``."""
    who = "distill_loss"
    code = _code(logits, "logits")
    xr, m, v, ld = _rows(logits, "logits")
    for name, t, dt in (("teacher_index", teacher_index, torch.int32), ("teacher_value", teacher_value, torch.float32)):
        if not isinstance(t, torch.Tensor) or t.dtype != dt:
            raise TypeError(f"{who}: {name} must be a {dt} tensor, got {getattr(t, 'dtype', type(t).__name__)}")
    shape = teacher_index.shape
    if not shape or shape[:-1] != logits.shape[:-1] or teacher_value.shape != shape:
        raise ValueError(f"{who}: teacher_index {tuple(shape)} and teacher_value {tuple(teacher_value.shape)} do not go with "
                         f"logits {tuple(logits.shape)}")
    k = shape[-1]
    if k > MAX_TEACHER_ENTRIES:
        raise ValueError(f"{who}: at most {MAX_TEACHER_ENTRIES} entries of the teacher per row, got {k}")
    ti = teacher_index if teacher_index.is_contiguous() else teacher_index.contiguous()
    tv = teacher_value if teacher_value.is_contiguous() else teacher_value.contiguous()
    y = _vector(labels, who, "labels", m, torch.int32)
    label_weight, weight, grad_scale = float(label_weight), float(weight), float(grad_scale)
    if not (weight - weight == 0.0 and label_weight - label_weight == 0.0):
        raise ValueError(f"{who}: weight and label_weight must be finite, got {weight} and {label_weight}")
    if label_weight != 0.0 and y is None:
        raise ValueError(f"{who}: label_weight needs labels")
    rs = _vector(row_scale, who, "row_scale", m, torch.float32)
    if logits.dim() > 2:
        _in_order(logits, who, labels=y, row_scale=rs)
    temperature = _temperature(temperature, who)
    dev = _device(logits, who, ti, tv, y, rs)
    if out is None:
        out = distill_output_like(logits, grad)
    loss = _result(out.loss, who, "loss", m, torch.float32, dev)
    dx = _result(out.dlogits, who, "dlogits", m * v, logits.dtype, dev) if grad else 0
    work = _scratch(out.work, who, _floats("distill_floats", m, v, code), dev)
    _launch(dev, lib().distill, xr.data_ptr(), ld, code, m, v, _ptr(ti) if k else 0, _ptr(tv) if k else 0, k, k, _ptr(y),
            temperature, weight, label_weight, _ptr(rs), grad_scale, loss, dx, v, work)
    return out if grad or out.dlogits is None else out._replace(dlogits=None)
