"""CPU checks of the operators on vocabulary rows: every refusal happens on the
host, before a device is used, and zero rows are a valid call."""
import ctypes

import pytest
import torch

from hikoboshi_b200 import HkbError, _lib, vocab


def refused(call, text, code=_lib.HKB_INVALID_ARGUMENT):
    with pytest.raises(HkbError) as e:
        call()
    assert e.value.code == code, e.value
    assert text in e.value.detail, e.value.detail


X, U = torch.zeros(3, 21), torch.zeros(3)
TV, TT = torch.zeros(3, 4), torch.zeros(3, 4, dtype=torch.int32)


@pytest.mark.parametrize("kwargs,text", [
    (dict(temperature=-0.5), "temperature"), (dict(temperature=float("nan")), "temperature"),
    (dict(temperature=float("inf")), "temperature"), (dict(temperature="1"), "number"),
    (dict(top_k=-1), "top_k"), (dict(top_k=1.5), "top_k"), (dict(top_k=True), "top_k"),
    (dict(top_p=1.5), "top_p"), (dict(top_p=-0.1), "top_p"), (dict(top_p=float("nan")), "top_p"),
    (dict(min_p=2.0), "min_p"), (dict(min_p=-1e-9), "min_p"),
    (dict(top_k=torch.zeros(3)), "int32"), (dict(top_p=torch.zeros(2)), "one number per row"),
    (dict(temperature=torch.zeros(3, dtype=torch.float64)), "float32"),
    (dict(min_p=torch.zeros(6)[::2]), "contiguous"),
])
def test_sample_settings_are_checked(kwargs, text):
    refused(lambda: vocab.sample_tokens(X, U, **kwargs), text)


@pytest.mark.parametrize("logits,text", [
    (torch.zeros(3, 21, dtype=torch.float64), "float32, float16 or bfloat16"),
    (torch.zeros(3, 21, dtype=torch.int32), "float32, float16 or bfloat16"),
    (torch.zeros(21, 3).t(), "stride 1"), (torch.zeros(3, 0), "at least one token"),
    (torch.tensor(1.0), "at least one token"), (None, "tensor"),
    (torch.zeros(4, 2, 21)[:, :1].expand(4, 3, 21), "one stride"),
    (torch.zeros(1, 262145), "HKB_VOCAB_MAX"),
])
def test_logits_are_checked(logits, text):
    u = torch.zeros(logits.shape[:-1]) if isinstance(logits, torch.Tensor) and logits.dim() else U
    refused(lambda: vocab.sample_tokens(logits, u), text)
    refused(lambda: vocab.top_logits(logits, 2), text)


def test_uniforms_are_checked():
    for u, text in ((torch.zeros(2), "one number per row"), (U.half(), "float32 or float64"),
                    (None, "tensor"), (torch.zeros(6)[::2], "contiguous")):
        refused(lambda: vocab.sample_tokens(X, u), text)


def test_top_is_checked():
    for k, text in ((0, "k must be 1"), (-3, "k must be 1"), (1025, "HKB_LISTING_MAX"),
                    (2**40, "HKB_LISTING_MAX"), (2.0, "whole number")):
        refused(lambda: vocab.top_logits(X, k), text)
    for t in (0.0, -1.0, 1e-31, 1e31, float("inf"), float("nan")):
        refused(lambda: vocab.top_logits(X, 3, temperature=t), "temperature")


@pytest.mark.parametrize("change,text", [
    (dict(values=TV.double()), "float32, float16 or bfloat16"), (dict(tokens=TT.long()), "int32"),
    (dict(tokens=TT[:, :3].contiguous()), "[.., k]"), (dict(values=TV[:2]), "[.., k]"),
    (dict(values=torch.zeros(4, 3).t()), "contiguous"),
    (dict(teacher_log_norm=torch.zeros(2)), "one number per row"),
    (dict(teacher_log_norm=U.double()), "float32"),
    (dict(temperature=0.0), "temperature"), (dict(temperature=float("nan")), "temperature"),
    (dict(temperature=1e-31), "temperature"), (dict(temperature=1e31), "temperature"),
    (dict(values=torch.zeros(3, 0), tokens=TT[:, :0]), "HKB_LISTING_MAX"),
    (dict(values=torch.zeros(3, 1025), tokens=torch.zeros(3, 1025, dtype=torch.int32)),
     "HKB_LISTING_MAX"),
])
def test_teacher_is_checked(change, text):
    kw = dict(values=TV, tokens=TT)
    kw.update(change)
    v, t = kw.pop("values"), kw.pop("tokens")
    refused(lambda: vocab.distill_loss(X, v, t, **kw), text)
    refused(lambda: vocab.distill_loss_and_grad(X, v, t, **kw), text)


@pytest.mark.parametrize("kwargs,text", [
    (dict(row_weights=torch.zeros(2)), "one number per row"),
    (dict(row_weights=U.double()), "float32"),
    (dict(grad_out=torch.zeros(3, 20)), "type and shape"),
    (dict(grad_out=torch.zeros(3, 21).half()), "type and shape"),
    (dict(grad_out=torch.zeros(21, 3).t()), "stride 1"),
    (dict(grad_out=torch.zeros(1, 21).expand(3, 21)), "must not overlap"),
])
def test_fused_outputs_are_checked(kwargs, text):
    refused(lambda: vocab.distill_loss_and_grad(X, TV, TT, **kwargs), text)


def test_gradient_lies_apart_from_what_else_is_read_and_written():
    x = torch.zeros(3, 21)
    tokens = torch.zeros(3, 21, dtype=torch.int32)
    # a student that is its own teacher, listed whole: the teacher's rows are the logits
    refused(lambda: vocab.distill_loss_and_grad(x, x, tokens, grad_out=x), "apart from the teacher")
    refused(lambda: vocab.distill_loss_and_grad(x, torch.ones(3, 21), tokens,
                                                grad_out=tokens.view(torch.float32)),
            "apart from the teacher")
    buf = torch.zeros(70)
    for name in ("row_weights", "teacher_log_norm"):
        refused(lambda: vocab.distill_loss_and_grad(x, torch.ones(3, 21), tokens,
                                                    grad_out=buf[:63].view(3, 21),
                                                    **{name: buf[62:65]}), "apart from the teacher")


def test_gradient_may_be_the_logits_but_not_overlap_them():
    buf = torch.zeros(4 * 21)
    x = buf[:63].view(3, 21)
    refused(lambda: vocab.distill_loss_and_grad(x, TV, TT, grad_out=buf[21:].view(3, 21)), "apart")
    refused(lambda: vocab.distill_loss_and_grad(x, TV, TT, grad_out=buf[1:64].view(3, 21)), "apart")
    if not torch.cuda.is_available():  # its own buffer passes the checks
        refused(lambda: vocab.distill_loss_and_grad(x, TV, TT, grad_out=x), "device",
                _lib.HKB_UNAVAILABLE)


def test_zero_rows_are_a_valid_call():
    x, u = torch.zeros(0, 21), torch.zeros(0)
    v, t = torch.zeros(0, 4), torch.zeros(0, 4, dtype=torch.int32)
    r = vocab.sample_tokens(x, u, top_k=3)
    assert r.tokens.shape == r.log_probs.shape == r.kept.shape == (0,)
    r = vocab.top_logits(torch.zeros(2, 0, 21), 5)
    assert r.values.shape == r.tokens.shape == (2, 0, 5) and r.log_norm.shape == (2, 0)
    loss, grad = vocab.distill_loss_and_grad(x, v, t)
    assert loss.shape == (0,) and grad.shape == (0, 21)
    xr = x.clone().requires_grad_()
    vocab.distill_loss(xr, v, t, teacher_log_norm=u).sum().backward()
    assert xr.grad.shape == (0, 21)


def test_null_pointers_are_refused():
    lib = _lib.load()
    rows = _lib.VocabRows(2, 21, _lib.F32, None, 21)
    assert lib.hkb_sample_tokens(0, None, None, None, None).code == 1
    assert lib.hkb_top_logits(0, None, 1, 1.0, None, None).code == 1
    assert lib.hkb_distill(0, None, None, None, None).code == 1
    assert lib.hkb_top_logits(0, ctypes.byref(rows), 1, 1.0, ctypes.byref(_lib.TopOut()), None
                              ).code == 1  # logits
    buf = (ctypes.c_float * 64)()
    rows.logits = ctypes.addressof(buf)
    for call in (lambda: lib.hkb_top_logits(0, ctypes.byref(rows), 1, 1.0,
                                            ctypes.byref(_lib.TopOut()), None),
                 lambda: lib.hkb_sample_tokens(0, ctypes.byref(rows),
                                               ctypes.byref(_lib.SampleSettings(top_p=1.0)),
                                               ctypes.byref(_lib.SampleOut()), None),
                 lambda: lib.hkb_distill(0, ctypes.byref(rows),
                                         ctypes.byref(_lib.DistillTeacher(k=1, temperature=1.0)),
                                         ctypes.byref(_lib.DistillOut()), None)):
        assert call().code == _lib.HKB_INVALID_ARGUMENT
    for field, value in (("rows", -1), ("rows", 2**28), ("vocab", 0), ("vocab", 262145),
                         ("dtype", _lib.F64), ("row_stride", -1)):
        bad = _lib.VocabRows(2, 21, _lib.F32, ctypes.addressof(buf), 21)
        setattr(bad, field, value)
        assert lib.hkb_top_logits(0, ctypes.byref(bad), 1, 1.0, ctypes.byref(_lib.TopOut()), None
                                  ).code == _lib.HKB_INVALID_ARGUMENT
    bad = _lib.VocabRows(2, 21, _lib.F32, ctypes.addressof(buf) + 2, 21)
    assert b"aligned" in lib.hkb_top_logits(0, ctypes.byref(bad), 1, 1.0,
                                            ctypes.byref(_lib.TopOut()), None).detail


def test_backward_entry_is_checked():
    lib = _lib.load()
    buf = (ctypes.c_float * 64)()
    at = ctypes.addressof(buf)
    rows = _lib.VocabRows(1, 21, _lib.F32, at, 21)
    t = _lib.DistillTeacher(k=1, temperature=1.0, values=at, tokens=at)
    for out, text in ((dict(loss=at, grad=at, stats=at), b"no loss"), (dict(grad=at), b"stats"),
                      (dict(stats=at), b"grad")):
        o = _lib.DistillOut(grad_row_stride=21, **out)
        st = lib.hkb_distill_backward(0, ctypes.byref(rows), ctypes.byref(t), ctypes.byref(o), None)
        assert st.code == _lib.HKB_INVALID_ARGUMENT and text in st.detail, st.detail
    rows.rows = 0
    o = _lib.DistillOut(grad_row_stride=21)
    assert lib.hkb_distill_backward(0, ctypes.byref(rows), ctypes.byref(t), ctypes.byref(o), None
                                    ).code == _lib.HKB_OK
