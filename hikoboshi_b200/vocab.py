"""Operators on vocabulary rows: torch front-end of ``hkb_sample_tokens``,
``hkb_top_logits`` and ``hkb_distill`` (include/hkb_mpnn.h).

A vocabulary row is one position's logits over V tokens: the [.., 21] rows of
:meth:`DesignEngine.score`, or any other model's.

* :func:`sample_tokens` draws a token of each row after temperature, top-k,
  top-p and min-p, from given uniforms;
* :func:`top_logits` takes each row's k largest logits in order and its
  log-sum-exp: a teacher's answer in the form that is stored;
* :func:`distill_loss` is the divergence of student rows from such answers, with
  its gradient by autograd; :func:`distill_loss_and_grad` gives loss and
  gradient in one pass over the rows.

Tensors are CUDA tensors of one device, logits f32, fp16 or bf16 with a last
dimension of stride 1 and leading dimensions that flatten to rows of one
stride; nothing is copied or converted on the way.  The work goes to torch's
current stream of that device, without synchronisation, workspaces or state.
Unfit arguments raise :class:`HkbError` with ``HKB_INVALID_ARGUMENT``.
"""
from __future__ import annotations

from ctypes import byref
from typing import NamedTuple

import torch

from . import _lib
from ._lib import HkbError, check

_DTYPES = {torch.float32: _lib.F32, torch.float16: _lib.F16, torch.bfloat16: _lib.BF16}
_FLOAT = (torch.float32,)
_INT = (torch.int32,)
_UNIFORMS = (torch.float32, torch.float64)


class SampledTokens(NamedTuple):
    tokens: torch.Tensor     # i32: the drawn token, -1 where none can be drawn
    log_probs: torch.Tensor  # f32: its log-probability among the kept tokens
    kept: torch.Tensor       # i32: how many tokens the filters kept


class TopLogits(NamedTuple):
    values: torch.Tensor     # [.., k] in the logits' type, largest first
    tokens: torch.Tensor     # [.., k] i32
    log_norm: torch.Tensor   # [..] f32: log sum exp(x / temperature)


def _invalid(why: str) -> HkbError:
    return HkbError(_lib.HKB_INVALID_ARGUMENT, why)


def _is_tensor(x, name: str) -> torch.Tensor:
    if not isinstance(x, torch.Tensor):
        raise _invalid(f"{name} must be a tensor")
    return x


def _rows(x: torch.Tensor, name: str = "logits"):
    """(rows, leading shape) of [.., V] logits, as the library takes them; never
    a copy."""
    _is_tensor(x, name)
    code = _DTYPES.get(x.dtype)
    if code is None:
        raise _invalid(f"{name} must be float32, float16 or bfloat16")
    shape = x.shape
    if len(shape) == 0 or shape[-1] == 0:
        raise _invalid(f"{name} must have a last dimension of at least one token")
    if x.layout is not torch.strided or x.is_neg():
        raise _invalid(f"{name} must be a plain strided tensor")
    v = shape[-1]
    stride = x.stride()
    if v > 1 and stride[-1] != 1:
        raise _invalid(f"{name} must have a last dimension of stride 1")
    if len(shape) == 2:
        n, step = shape[0], stride[0]
    else:
        n, step = _flatten(shape[:-1], stride[:-1])
        if step is None:
            raise _invalid(f"{name}: the leading dimensions must flatten to rows of one stride")
    return _lib.VocabRows(n, v if v < 2**31 else 2**31 - 1, code, x.data_ptr(),
                          step if n > 1 else v), shape[:-1]


def _flatten(shape, stride):
    """(number, stride) of the dimensions taken as one, stride None if they
    have no common one."""
    n, step = 1, 0
    for size, st in zip(reversed(shape), reversed(stride)):
        if size == 1:
            continue
        if n == 1:
            step = st
        elif size and n and st != step * n:
            step = None
            break
        n *= size
    n = 1
    for size in shape:
        n *= size
    return (n, step) if n else (0, 0)


def _vector(x, lead, device, dtypes, name) -> torch.Tensor:
    """A dense per-row tensor of the leading shape."""
    _is_tensor(x, name)
    if x.device != device:
        raise _invalid(f"{name} must be on the logits' device")
    if x.dtype not in dtypes:
        raise _invalid(f"{name} must be " + " or ".join(str(d).split(".")[1] for d in dtypes))
    if x.shape != lead:
        raise _invalid(f"{name} must have one number per row")
    if not x.is_contiguous() or x.is_neg():
        raise _invalid(f"{name} must be contiguous")
    return x


# the current stream's handle without a Stream object around it
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda index: torch.cuda.current_stream(index).cuda_stream)


def _call(fn, device: torch.device, *args) -> None:
    if device.type == "cuda":
        st = fn(device.index, *args, _raw_stream(device.index))
        if st.code:
            check(st)
        return
    # the library checks the other arguments first, then refuses the device
    st = fn(-1, *args, None)
    if st.code == _lib.HKB_INVALID_ARGUMENT and st.detail == b"device ordinal out of range":
        raise _invalid("logits must be on a CUDA device")
    check(st)


def _number(v, name: str) -> float:
    if isinstance(v, bool) or not isinstance(v, (int, float)):
        raise _invalid(f"{name} must be a number or a tensor of one number per row")
    return float(v)


def sample_tokens(logits, uniforms, *, temperature=1.0, top_k=0, top_p=1.0,
                  min_p=0.0) -> SampledTokens:
    """Draws one token of each row of ``logits`` [.., V] with ``uniforms`` [..]
    (f32 or f64 in [0, 1]).

    The tokens, in the order (logit down, index up), are cut to the shortest of
    three heads: the first ``top_k`` (0 = off); the shortest whose mass reaches
    ``top_p`` of the top-k mass (1 = off; at least one token); those of at
    least ``min_p`` times the largest probability (0 = off).  The token is the
    first in index order whose running kept mass exceeds u times the kept
    mass.  ``temperature`` 0 takes the largest logit.

    Each setting is a number, or a tensor [..] with a setting per row (f32,
    ``top_k`` i32).  Rows whose tensor settings or uniforms are out of range
    give token -1, log_prob NaN and kept 0; rows with no logit above -inf give
    -1, -inf and 0.  A NaN logit counts as -inf.
    """
    rows, lead = _rows(logits)
    device = logits.device
    u = _vector(uniforms, lead, device, _UNIFORMS, "uniforms")
    s = _lib.SampleSettings()
    s.uniforms = u.data_ptr()
    s.uniforms_dtype = _lib.F64 if u.dtype == torch.float64 else _lib.F32
    if isinstance(temperature, torch.Tensor):
        s.temperatures = _vector(temperature, lead, device, _FLOAT, "temperature").data_ptr()
    else:
        s.temperature = _number(temperature, "temperature")
    if isinstance(top_k, torch.Tensor):
        s.top_ks = _vector(top_k, lead, device, _INT, "top_k").data_ptr()
    elif isinstance(top_k, bool) or not isinstance(top_k, int):
        raise _invalid("top_k must be a whole number or a tensor of one per row")
    else:
        s.top_k = max(-1, min(top_k, 2**31 - 1))
    if isinstance(top_p, torch.Tensor):
        s.top_ps = _vector(top_p, lead, device, _FLOAT, "top_p").data_ptr()
    else:
        s.top_p = _number(top_p, "top_p")
    if isinstance(min_p, torch.Tensor):
        s.min_ps = _vector(min_p, lead, device, _FLOAT, "min_p").data_ptr()
    else:
        s.min_p = _number(min_p, "min_p")
    tokens = logits.new_empty(lead, dtype=torch.int32)
    log_probs = logits.new_empty(lead, dtype=torch.float32)
    kept = logits.new_empty(lead, dtype=torch.int32)
    o = _lib.SampleOut(tokens.data_ptr(), log_probs.data_ptr(), kept.data_ptr())
    _call(_lib.load().hkb_sample_tokens, device, byref(rows), byref(s), byref(o))
    return SampledTokens(tokens, log_probs, kept)


def top_logits(logits, k: int, *, temperature: float = 1.0) -> TopLogits:
    """The ``k`` largest logits of each row of ``logits`` [.., V] with their
    tokens, in the order (logit down, index up), and log sum exp(x / temperature).
    Places past a row's logits above -inf hold (-inf, -1); a NaN logit counts
    as -inf."""
    rows, lead = _rows(logits)
    if isinstance(k, bool) or not isinstance(k, int):
        raise _invalid("k must be a whole number")
    k = max(-1, min(k, 2**31 - 1))
    n = max(0, min(k, _lib.LISTING_MAX))
    device = logits.device
    values = logits.new_empty((*lead, n), dtype=logits.dtype)
    tokens = logits.new_empty((*lead, n), dtype=torch.int32)
    log_norm = logits.new_empty(lead, dtype=torch.float32)
    o = _lib.TopOut(values.data_ptr(), tokens.data_ptr(), log_norm.data_ptr())
    _call(_lib.load().hkb_top_logits, device, byref(rows), k,
          _number(temperature, "temperature"), byref(o))
    return TopLogits(values, tokens, log_norm)


def _teacher(lead, device, values, tokens, log_norm, temperature) -> _lib.DistillTeacher:
    _is_tensor(values, "teacher_values")
    _is_tensor(tokens, "teacher_tokens")
    code = _DTYPES.get(values.dtype)
    if code is None:
        raise _invalid("teacher_values must be float32, float16 or bfloat16")
    if tokens.dtype is not torch.int32:
        raise _invalid("teacher_tokens must be int32")
    shape = values.shape
    if len(shape) == 0 or shape[:-1] != lead or tokens.shape != shape:
        raise _invalid("teacher_values and teacher_tokens must be [.., k] with the logits' rows")
    if values.device != device:
        raise _invalid("teacher_values must be on the logits' device")
    if tokens.device != device:
        raise _invalid("teacher_tokens must be on the logits' device")
    if not values.is_contiguous() or not tokens.is_contiguous() or values.is_neg():
        raise _invalid("teacher_values and teacher_tokens must be contiguous")
    if log_norm is not None:
        log_norm = _vector(log_norm, lead, device, _FLOAT, "teacher_log_norm").data_ptr()
    return _lib.DistillTeacher(min(shape[-1], 2**31 - 1), code, values.data_ptr(),
                               tokens.data_ptr(), log_norm, _number(temperature, "temperature"))


def _weights(w, lead, device):
    """(pointer, stride) of per-row weights: one stride, 0 where broadcast."""
    if w is None:
        return None, 0
    _is_tensor(w, "row_weights")
    if w.device != device:
        raise _invalid("row_weights must be on the logits' device")
    if w.dtype is not torch.float32:
        raise _invalid("row_weights must be float32")
    if w.shape != lead:
        raise _invalid("row_weights must have one number per row")
    _, step = _flatten(w.shape, w.stride())
    if step is None or w.is_neg():
        raise _invalid("row_weights must flatten to one stride")
    return w.data_ptr(), step


def _backward(logits, values, tokens, log_norm, temperature, grad_loss):
    rows, lead = _rows(logits)
    device = logits.device
    t = _teacher(lead, device, values, tokens, log_norm, temperature)
    grad = logits.new_empty(logits.shape)
    if rows.rows:
        _, step = _flatten(grad_loss.shape, grad_loss.stride())
        if step is None or grad_loss.is_neg():
            grad_loss = grad_loss.clone(memory_format=torch.contiguous_format).resolve_neg()
        pointer, step = _weights(grad_loss, lead, device)
        o = _lib.DistillOut(None, grad.data_ptr(), logits.shape[-1], pointer, step)
        _call(_lib.load().hkb_distill, device, byref(rows), byref(t), byref(o))
    return grad


def _forward(logits, values, tokens, log_norm, temperature):
    rows, lead = _rows(logits)
    device = logits.device
    t = _teacher(lead, device, values, tokens, log_norm, temperature)
    loss = logits.new_empty(lead, dtype=torch.float32)
    o = _lib.DistillOut(loss.data_ptr(), None, 0, None, 0)
    _call(_lib.load().hkb_distill, device, byref(rows), byref(t), byref(o))
    return loss


class _DistillLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, values, tokens, log_norm, temperature):
        ctx.save_for_backward(logits, values, tokens, log_norm)
        ctx.temperature = temperature
        return _forward(logits, values, tokens, log_norm, temperature)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_loss):
        return _backward(*ctx.saved_tensors, ctx.temperature, grad_loss), None, None, None, None


def distill_loss(logits, teacher_values, teacher_tokens, *, teacher_log_norm=None,
                 temperature: float = 1.0) -> torch.Tensor:
    """Divergence [..] (f32) of the rows of ``logits`` [.., V] from a teacher's
    listed logits ``teacher_values`` [.., k] at ``teacher_tokens`` [.., k] (i32),
    differentiable with respect to ``logits``.

    Without ``teacher_log_norm`` the teacher is softmax(values / temperature)
    over the list and the loss temperature^2 KL(teacher || student).  With it
    (:class:`TopLogits`.log_norm at the same temperature) the listed tokens keep
    their true masses and all others form one class with what is left, against
    the student's mass outside the list.  A negative token or a value of -inf is
    no entry; a row without entries has loss and gradient 0 whatever its logits.
    A token >= V makes its row NaN.

    The backward pass reads ``logits`` again, so they must not be overwritten
    before it.  Autograd through this call cannot be captured into a CUDA
    graph (an eager graph of the same leaves would break the capture): there
    it raises HKB_FAILED_PRECONDITION; capture :func:`distill_loss_and_grad`.
    """
    if not (isinstance(logits, torch.Tensor) and logits.requires_grad
            and torch.is_grad_enabled()):
        return _forward(logits, teacher_values, teacher_tokens, teacher_log_norm, temperature)
    if logits.is_cuda and torch.cuda.is_current_stream_capturing():
        raise HkbError(_lib.HKB_FAILED_PRECONDITION,
                       "autograd through distill_loss cannot be captured; capture "
                       "distill_loss_and_grad")
    return _DistillLoss.apply(logits, teacher_values, teacher_tokens, teacher_log_norm,
                              temperature)


def distill_loss_and_grad(logits, teacher_values, teacher_tokens, *, teacher_log_norm=None,
                          temperature: float = 1.0, row_weights=None, grad_out=None):
    """(loss [..], gradient [.., V]) of :func:`distill_loss` in one pass over the
    rows: the gradient of ``sum(row_weights * loss)`` with respect to ``logits``
    (weights 1 by default), in the logits' type.  A row of weight 0 has gradient
    0.  ``grad_out`` receives the gradient and may be ``logits`` itself, whose
    memory the gradient then takes; autograd does not see this call."""
    rows, lead = _rows(logits)
    device = logits.device
    t = _teacher(lead, device, teacher_values, teacher_tokens, teacher_log_norm, temperature)
    pointer, step = _weights(row_weights, lead, device)
    if grad_out is None:
        grad_out = logits.new_empty(logits.shape)
        grad_stride = logits.shape[-1]
    else:
        _is_tensor(grad_out, "grad_out")
        if grad_out.device != device:
            raise _invalid("grad_out must be on the logits' device")
        if grad_out.dtype is not logits.dtype or grad_out.shape != logits.shape:
            raise _invalid("grad_out must have the logits' type and shape")
        grad_stride = _rows(grad_out, "grad_out")[0].row_stride
    loss = logits.new_empty(lead, dtype=torch.float32)
    o = _lib.DistillOut(loss.data_ptr(), grad_out.data_ptr(), grad_stride, pointer, step)
    _call(_lib.load().hkb_distill, device, byref(rows), byref(t), byref(o))
    return loss, grad_out


__all__ = ["SampledTokens", "TopLogits", "distill_loss", "distill_loss_and_grad",
           "sample_tokens", "top_logits"]
