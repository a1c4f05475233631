"""The distillation loss and its gradient keep their digits over the whole range
of temperatures: the loss stays of the order of the logits' variance while the
divergence falls with temperature^2.  On a B200, against the definition in 80
bits; the bounds are small beside what they bound."""
import numpy as np
import pytest
import torch

from hikoboshi_b200 import HkbError
from test_gpu_vocab import gen, logits, teacher
from vocab_reference import STEP, TINY, to64

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
LD = np.longdouble


@pytest.fixture(scope="module")
def vocab():
    from hikoboshi_b200 import vocab
    return vocab


def reference(x, values, tokens, norm, tau):
    """Loss, gradient and the weights' exponents of one row, tokens listed once."""
    x, values, tau = x.astype(LD), values.astype(LD), LD(tau)
    z = (x - x.max()) / tau
    log_p = z - np.log(np.exp(z).sum())
    p = np.exp(log_p)
    a = values / tau
    if norm is None:
        log_q = a - a.max()
        log_q -= np.log(np.exp(log_q).sum())
    else:
        log_q = a - LD(norm)
    q = np.exp(log_q)
    loss = (q * (log_q - log_p[tokens])).sum()
    target = np.zeros_like(p)
    target[tokens] = q
    mass = q.sum()
    if norm is not None and len(tokens) < len(x):
        off = np.ones(len(x), bool)
        off[tokens] = False
        rest_q, rest_p = max(LD(0), 1 - q.sum()), p[off].sum()
        if rest_q > 0:
            loss += rest_q * np.log(rest_q / rest_p)
            target[off] = rest_q * p[off] / rest_p
        mass = q.sum() + rest_q
    return loss * tau * tau, tau * (mass * p - target), p, target, z


def bounds(size, loss, grad, p, target, z, tau, dtype):
    """Of the loss's and the gradient's error above the temperature from which
    the sums are 64-bit: a thread adds at most 256 weights one after another and
    joins them with 31 others', a weight is off by 4 roundings; the loss adds
    terms of up to ln(size) + 1; 64 of them one after another.  The
    gradient's factor takes 32-bit rounding only where nothing cancels any more."""
    sums = 2.0 ** -53 * (256 + 32 + 4)
    loss_err = tau * tau * (2 * sums + 2.0 ** -53 * 96 * (1 + np.log(size))) + 2.0 ** -24 * abs(loss)
    grad_err = tau * (p + target) * 2 * sums + 2.0 ** -24 * (3 * -z + 8) * abs(grad)
    return loss_err, grad_err + STEP[dtype] * (abs(grad) + grad_err) + TINY[dtype]


def check(got, x, v, t, norm, tau, dtype, w):
    loss, grad = to64(got[0]), to64(got[1])
    for r in range(len(x)):
        want, g, p, target, z = reference(to64(x[r]), to64(v[r]), t[r].long().cpu().numpy(),
                                          None if norm is None else float(norm[r]), tau)
        loss_err, grad_err = bounds(x.shape[1], want, g, p, target, z, tau, dtype)
        # a bound that says something
        assert loss_err <= 0.05 * abs(want), (r, tau, loss_err, want)
        if dtype == F32:
            assert grad_err.max() <= 0.05 * abs(g).max()
        assert abs(loss[r] - want) <= loss_err, (r, tau, loss[r], want, loss_err)
        off = abs(grad[r] - w * g)
        assert (off <= grad_err).all(), (r, tau, off.argmax(), off.max(), grad_err[off.argmax()])


# a thread a row; one CTA and a cluster; a CTA that streams; teams of 4 and of 8 lanes
ROWS = [(7, 8), (150, 21), (7, 32), (7, 500), (7, 5000), (7, 40000), (700, 900), (650, 20000),
        (9500, 100), (4800, 800)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,size", ROWS)
def test_hot_distillation_keeps_its_digits(vocab, rows, size, dtype):
    at = torch.tensor([0, 1, rows // 2, rows - 1], device="cuda").unique()
    for tau in (16.5, 30.0, 100.0, 1e3, 1e4):
        for tail in (False, True):
            for k in sorted({min(size, max(5, size // 100)), min(size, 100)}):
                x = logits(rows, size, dtype, size + k)
                v, t, norm = teacher(x, k, F32, k, tau, tail)
                w = torch.full((rows,), 0.75, device="cuda")
                kw = dict(teacher_log_norm=norm, temperature=tau)
                got = vocab.distill_loss_and_grad(x, v, t, row_weights=w, **kw)
                check([a[at] for a in got], x[at], v[at], t[at], norm[at] if tail else None,
                      float(np.float32(tau)), dtype, 0.75)
                z = x.clone().requires_grad_()
                l2 = vocab.distill_loss(z, v, t, **kw)
                (g2,) = torch.autograd.grad(l2, z, w)
                assert torch.equal(l2.detach(), got[0]) and torch.equal(g2, got[1])
                y = x.clone()
                vocab.distill_loss_and_grad(y, v, t, row_weights=w, grad_out=y, **kw)
                assert torch.equal(y, got[1])


@pytest.mark.gpu
@pytest.mark.parametrize("rows,size", ROWS)
def test_hot_rows_with_masks_and_no_numbers(vocab, rows, size):
    x = logits(rows, size, F32, 3)
    v, t, norm = teacher(x, 6, F32, 4, 50.0, True)
    x[0] = -float("inf")
    x[1, 5] = float("nan")
    x[2, 7] = float("inf")
    x[3, ::2] = -float("inf")
    x[3].scatter_(0, t[3].long(), 1.0)
    x[4] = torch.finfo(F32).min
    x[4, 3] = torch.finfo(F32).max
    t[5] = -1
    for n in (None, norm):
        loss, grad = vocab.distill_loss_and_grad(x, v, t, teacher_log_norm=n, temperature=50.0)
        assert loss[:3].isnan().all() and grad[:3].isnan().all()
        assert loss[5] == 0 and (grad[5] == 0).all()
        assert loss[3].isfinite() and (grad[3][x[3] == -float("inf")] == 0).all()
        assert not grad[4].isnan().any() and loss[4] > 0
        check((loss[6:7], grad[6:7]), x[6:7], v[6:7], t[6:7], None if n is None else n[6:7], 50.0,
              F32, 1.0)


@pytest.mark.gpu
def test_both_sides_of_the_change_to_64_bits_agree(vocab):
    # the same loss to what 32 bits leave of it at that temperature
    for rows, size in ROWS:
        x = logits(rows, size, F32, 5)
        lo, hi = 16.0, float(np.nextafter(np.float32(16.0), np.float32(17.0)))
        v, t, norm = teacher(x, min(size, 9), F32, 6, lo, True)
        for n in (None, norm):
            a = vocab.distill_loss_and_grad(x, v, t, teacher_log_norm=n, temperature=lo)
            b = vocab.distill_loss_and_grad(x, v, t, teacher_log_norm=n, temperature=hi)
            # 2^-24 a rounding; up to 160 weights added one after another, and a
            # change of 2^-23 of the temperature itself
            assert (a[0] - b[0]).abs().max() <= 16 ** 2 * 180 * 2.0 ** -24 + 1e-6 * a[0].abs().max()
            assert (a[1] - b[1]).abs().max() <= 16 * 180 * 2.0 ** -24


def test_temperatures_past_the_last_are_refused():
    from hikoboshi_b200 import vocab
    x, v = torch.zeros(3, 21), torch.zeros(3, 4)
    t = torch.zeros(3, 4, dtype=torch.int32)
    for tau in (1.0001e4, 1e5, 1e30):
        for call in (vocab.distill_loss, vocab.distill_loss_and_grad):
            with pytest.raises(HkbError) as e:
                call(x, v, t, temperature=tau)
            assert e.value.code == 1 and "1e4" in e.value.detail
    with pytest.raises(HkbError) as e:  # a log-norm has no such loss
        vocab.top_logits(x, 3, temperature=1e30)
    assert "temperature" not in e.value.detail
