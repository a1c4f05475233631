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

import ctypes
import math
from typing import NamedTuple

import torch

from . import _lib
from ._lib import HkbError, check

_DTYPES = {torch.float32: _lib.F32, torch.float16: _lib.F16, torch.bfloat16: _lib.BF16}


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
    """(2-d view, leading shape) of [.., V] logits; never a copy."""
    _is_tensor(x, name)
    if x.dtype not in _DTYPES:
        raise _invalid(f"{name} must be float32, float16 or bfloat16")
    if x.dim() == 0 or x.shape[-1] == 0:
        raise _invalid(f"{name} must have a last dimension of at least one token")
    if x.layout != torch.strided or x.is_conj() or x.is_neg():
        raise _invalid(f"{name} must be a plain strided tensor")
    lead = x.shape[:-1]
    if x.dim() == 1:
        x = x.unsqueeze(0)
    if x.shape[-1] > 1 and x.stride(-1) != 1:
        raise _invalid(f"{name} must have a last dimension of stride 1")
    if x.dim() > 2:
        try:
            x = x.view(-1, x.shape[-1]) if x.numel() else x.reshape(0, x.shape[-1])
        except RuntimeError:
            raise _invalid(f"{name}: the leading dimensions must flatten to rows of one stride")
    return x, lead


def _struct_rows(x: torch.Tensor) -> _lib.VocabRows:
    stride = x.stride(0) if x.shape[0] > 1 else x.shape[1]
    return _lib.VocabRows(x.shape[0], min(x.shape[1], 2**31 - 1), _DTYPES[x.dtype], x.data_ptr(),
                          stride)


def _on(x: torch.Tensor, like: torch.Tensor, name: str) -> None:
    if x.device != like.device:
        raise _invalid(f"{name} must be on the logits' device")


def _vector(x, lead, like, dtypes, name) -> torch.Tensor:
    """A dense per-row tensor of the leading shape."""
    _is_tensor(x, name)
    _on(x, like, name)
    if x.dtype not in dtypes:
        raise _invalid(f"{name} must be " + " or ".join(str(d).split(".")[1] for d in dtypes))
    if x.shape != lead:
        raise _invalid(f"{name} must have one number per row")
    if not x.is_contiguous():
        raise _invalid(f"{name} must be contiguous")
    return x


def _call(fn, x: torch.Tensor, *args) -> None:
    if x.device.type != "cuda":
        # the library checks the other arguments first, then refuses the device
        st = fn(-1, *args, None)
        if st.code == _lib.HKB_INVALID_ARGUMENT and st.detail == b"device ordinal out of range":
            raise _invalid("logits must be on a CUDA device")
        check(st)
        return
    stream = torch.cuda.current_stream(x.device).cuda_stream
    check(fn(x.device.index, *args, ctypes.c_void_p(stream)))


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
    x, lead = _rows(logits)
    u = _vector(uniforms, lead, x, (torch.float32, torch.float64), "uniforms")
    s = _lib.SampleSettings()
    hold = []
    for name, v, dtype in (("temperature", temperature, torch.float32),
                           ("top_k", top_k, torch.int32), ("top_p", top_p, torch.float32),
                           ("min_p", min_p, torch.float32)):
        if isinstance(v, torch.Tensor):
            hold.append(_vector(v, lead, x, (dtype,), name))
            setattr(s, name + "s" if name != "temperature" else "temperatures", v.data_ptr())
        elif name == "top_k":
            if isinstance(v, bool) or not isinstance(v, int):
                raise _invalid("top_k must be a whole number or a tensor of one per row")
            s.top_k = max(-1, min(v, 2**31 - 1))
        else:
            setattr(s, name, _number(v, name))
    s.uniforms = u.data_ptr()
    s.uniforms_dtype = _lib.F64 if u.dtype == torch.float64 else _lib.F32
    out = SampledTokens(torch.empty(lead, dtype=torch.int32, device=x.device),
                        torch.empty(lead, dtype=torch.float32, device=x.device),
                        torch.empty(lead, dtype=torch.int32, device=x.device))
    rows = _struct_rows(x)
    o = _lib.SampleOut(out.tokens.data_ptr(), out.log_probs.data_ptr(), out.kept.data_ptr())
    _call(_lib.load().hkb_sample_tokens, x, ctypes.byref(rows), ctypes.byref(s), ctypes.byref(o))
    return out


def top_logits(logits, k: int, *, temperature: float = 1.0) -> TopLogits:
    """The ``k`` largest logits of each row of ``logits`` [.., V] with their
    tokens, in the order (logit down, index up), and log sum exp(x / temperature).
    Places past a row's logits above -inf hold (-inf, -1); a NaN logit counts
    as -inf."""
    x, lead = _rows(logits)
    if isinstance(k, bool) or not isinstance(k, int):
        raise _invalid("k must be a whole number")
    k = max(-1, min(k, 2**31 - 1))
    n = max(0, min(k, _lib.LISTING_MAX))
    out = TopLogits(torch.empty((*lead, n), dtype=x.dtype, device=x.device),
                    torch.empty((*lead, n), dtype=torch.int32, device=x.device),
                    torch.empty(lead, dtype=torch.float32, device=x.device))
    rows = _struct_rows(x)
    o = _lib.TopOut(out.values.data_ptr(), out.tokens.data_ptr(), out.log_norm.data_ptr())
    _call(_lib.load().hkb_top_logits, x, ctypes.byref(rows), k,
          _number(temperature, "temperature"), ctypes.byref(o))
    return out


def _teacher(x, lead, values, tokens, log_norm, temperature) -> _lib.DistillTeacher:
    _is_tensor(values, "teacher_values")
    _is_tensor(tokens, "teacher_tokens")
    if values.dtype not in _DTYPES:
        raise _invalid("teacher_values must be float32, float16 or bfloat16")
    if tokens.dtype != torch.int32:
        raise _invalid("teacher_tokens must be int32")
    if values.dim() == 0 or values.shape[:-1] != lead or tokens.shape != values.shape:
        raise _invalid("teacher_values and teacher_tokens must be [.., k] with the logits' rows")
    _on(values, x, "teacher_values")
    _on(tokens, x, "teacher_tokens")
    if not values.is_contiguous() or not tokens.is_contiguous():
        raise _invalid("teacher_values and teacher_tokens must be contiguous")
    t = _lib.DistillTeacher()
    t.k = min(values.shape[-1], 2**31 - 1)
    t.dtype = _DTYPES[values.dtype]
    t.values = values.data_ptr()
    t.tokens = tokens.data_ptr()
    if log_norm is not None:
        t.log_norm = _vector(log_norm, lead, x, (torch.float32,), "teacher_log_norm").data_ptr()
        if t.log_norm is None:  # no rows: keep the form of the loss
            t.log_norm = 0
    t.temperature = _number(temperature, "temperature")
    return t


def _weights(w, lead, x):
    """(pointer, stride) of per-row weights: one stride, 0 where broadcast."""
    if w is None:
        return None, 0
    _is_tensor(w, "row_weights")
    _on(w, x, "row_weights")
    if w.dtype != torch.float32:
        raise _invalid("row_weights must be float32")
    if w.shape != lead:
        raise _invalid("row_weights must have one number per row")
    if w.numel() and all(s == 0 or n == 1 for s, n in zip(w.stride(), w.shape)):
        return w.data_ptr(), 0
    if w.dim() <= 1:
        return w.data_ptr(), w.stride(0) if w.dim() else 0
    try:
        return w.data_ptr(), w.view(-1).stride(0)
    except RuntimeError:
        raise _invalid("row_weights must flatten to one stride")


def _distill(x, teacher, loss, grad, weights) -> None:
    rows = _struct_rows(x)
    o = _lib.DistillOut()
    if loss is not None:
        o.loss = loss.data_ptr()
    if grad is not None:
        o.grad = grad.data_ptr()
        o.grad_row_stride = grad.stride(0) if grad.shape[0] > 1 else grad.shape[1]
    o.row_weights, o.row_weight_stride = weights
    _call(_lib.load().hkb_distill, x, ctypes.byref(rows), ctypes.byref(teacher), ctypes.byref(o))


class _DistillLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, values, tokens, log_norm, temperature):
        x, lead = _rows(logits)
        t = _teacher(x, lead, values, tokens, log_norm, temperature)
        loss = torch.empty(lead, dtype=torch.float32, device=x.device)
        if x.shape[0]:
            _distill(x, t, loss, None, (None, 0))
        ctx.save_for_backward(logits, values, tokens, log_norm)
        ctx.temperature = temperature
        return loss

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_loss):
        logits, values, tokens, log_norm = ctx.saved_tensors
        x, lead = _rows(logits)
        t = _teacher(x, lead, values, tokens, log_norm, ctx.temperature)
        grad = torch.empty(logits.shape, dtype=x.dtype, device=x.device)
        if x.shape[0]:
            try:
                w = _weights(grad_loss, lead, x)
            except HkbError:
                grad_loss = grad_loss.contiguous()
                w = _weights(grad_loss, lead, x)
            _distill(x, t, None, grad.view(x.shape), w)
        return grad, None, None, None, None


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
    _rows(logits)
    if (torch.is_grad_enabled() and logits.requires_grad and logits.is_cuda
            and torch.cuda.is_current_stream_capturing()):
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
    x, lead = _rows(logits)
    x = x.detach()
    t = _teacher(x, lead, teacher_values, teacher_tokens, teacher_log_norm, temperature)
    w = _weights(row_weights, lead, x)
    loss = torch.empty(lead, dtype=torch.float32, device=x.device)
    if grad_out is None:
        grad_out = torch.empty(logits.shape, dtype=x.dtype, device=x.device)
    else:
        _is_tensor(grad_out, "grad_out")
        _on(grad_out, x, "grad_out")
        if grad_out.dtype != x.dtype or grad_out.shape != logits.shape:
            raise _invalid("grad_out must have the logits' type and shape")
    g, _ = _rows(grad_out.detach(), "grad_out")
    _distill(x, t, loss, g, w)
    return loss, grad_out


__all__ = ["SampledTokens", "TopLogits", "distill_loss", "distill_loss_and_grad",
           "sample_tokens", "top_logits"]
