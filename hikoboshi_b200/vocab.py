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

Of all results only :func:`distill_loss` is differentiable, and with respect to
``logits`` alone: a teacher's tensors are constants, and what the other functions
return is detached, also from logits that require grad.  The functions are not
registered torch operators: ``torch.func`` transforms and
``torch.compile(fullgraph=True)`` raise, ``torch.compile`` without it calls them
between its graphs, and tracers of dispatched operators (``torch.export``,
``make_fx``) must not be used on them.
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from . import _lib

_lib.load()  # the operators' library, which the module below calls
try:
    from . import _vocab
except ImportError as e:
    raise ImportError("hikoboshi_b200/_vocab.so is not built for this torch; run "
                      "__graft_entry__.build() (or python hikoboshi_b200/_build.py)") from e


class SampledTokens(NamedTuple):
    tokens: torch.Tensor     # i32: the drawn token, -1 where none can be drawn
    log_probs: torch.Tensor  # f32: its log-probability among the kept tokens
    kept: torch.Tensor       # i32: how many tokens the filters kept


class TopLogits(NamedTuple):
    values: torch.Tensor     # [.., k] in the logits' type, largest first
    tokens: torch.Tensor     # [.., k] i32
    log_norm: torch.Tensor   # [..] f32: log sum exp(x / temperature)


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
    -1, -inf and 0.  A NaN logit counts as -inf.  Not differentiable.
    """
    return SampledTokens(*_vocab.sample(logits, uniforms, temperature, top_k, top_p, min_p))


def top_logits(logits, k: int, *, temperature: float = 1.0) -> TopLogits:
    """The ``k`` largest logits of each row of ``logits`` [.., V] with their
    tokens, in the order (logit down, index up), and log sum exp(x / temperature).
    Places past a row's logits above -inf hold (-inf, -1); a NaN logit counts
    as -inf.  ``temperature`` is 1e-30 to 1e30.  Not differentiable."""
    return TopLogits(*_vocab.top(logits, k, temperature))


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
    A token >= V makes its row NaN, and so do an entry's value that is NaN or +inf,
    a log-norm that is not finite, a NaN or +inf logit, and a row of logits without
    one above -inf.  ``temperature`` is 1e-30 to 1e4; up to 16 the student's
    sums are 32-bit and the loss is off by up to 2e-7 temperature^2, above that
    they are 64-bit.

    The loss is differentiable once, backwards; logits with a forward-mode tangent
    are refused.  The backward pass reads ``logits`` and the
    teacher's tensors again, so they must not be overwritten before it.
    Autograd through this call cannot be captured into a CUDA graph (an eager
    graph of the same leaves would break the capture): there it raises
    HKB_FAILED_PRECONDITION, a backward pass alone RuntimeError; capture
    :func:`distill_loss_and_grad`.
    """
    return _vocab.loss(logits, teacher_values, teacher_tokens, teacher_log_norm, temperature)


def distill_loss_and_grad(logits, teacher_values, teacher_tokens, *, teacher_log_norm=None,
                          temperature: float = 1.0, row_weights=None, grad_out=None):
    """(loss [..], gradient [.., V]) of :func:`distill_loss` in one pass over the
    rows: the gradient of ``sum(row_weights * loss)`` with respect to ``logits``
    (weights 1 by default), in the logits' type.  A row of weight 0 has gradient
    0.  ``grad_out`` receives the gradient and may be ``logits`` itself, whose
    memory the gradient then takes; it lies apart from all other arguments.
    Autograd does not record this call, but counts it as a change of
    ``grad_out``."""
    return _vocab.loss_and_grad(logits, teacher_values, teacher_tokens, teacher_log_norm,
                                temperature, row_weights, grad_out)


__all__ = ["SampledTokens", "TopLogits", "distill_loss", "distill_loss_and_grad",
           "sample_tokens", "top_logits"]
