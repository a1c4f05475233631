"""Every entry of the distillation gradient on rows that masks, listings and large
logits make special: where it is a number it lies within the bound, and it is NaN
exactly where the definition is.  On a B200, all kernels."""
import numpy as np
import pytest
import torch

from test_gpu_vocab import logits, teacher
from vocab_reference import distill_row, to64

pytestmark = pytest.mark.gpu

INF = float("inf")
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


@pytest.fixture(scope="module")
def vocab():
    from hikoboshi_b200 import vocab
    return vocab


def check_every_entry(loss, grad, x, values, tokens, norm, tau, weights):
    """Of rows whose definition has no NaN in places only."""
    l64, g64, x64, v64, w64 = (to64(a) for a in (loss, grad, x, values, weights))
    t64 = tokens.cpu().numpy()
    for r in range(len(x64)):
        with np.errstate(invalid="ignore", divide="ignore"):
            want, g, lerr, gerr = distill_row(x64[r], v64[r], t64[r],
                                              None if norm is None else float(norm[r]), tau,
                                              x.dtype)
        if len(g) <= 32:
            # short rows hold a token's mass in 32 bits: each entry's is rounded and
            # added (half a step of 2^-24 each), then the mass times a rounded factor
            # and the product's rounding, 2^-24 each, of temperature * mass
            ok = (t64[r] >= 0) & (t64[r] < len(g)) & (v64[r] > -INF)
            a = v64[r][ok] / tau
            q = np.exp(a - (np.logaddexp.reduce(a) if norm is None else float(norm[r])))
            mass, entries = np.zeros(len(g)), np.zeros(len(g))
            np.add.at(mass, t64[r][ok], q)
            np.add.at(entries, t64[r][ok], 1)
            gerr = gerr + 2.0 ** -24 * (2 * entries + 2) * tau * mass
        assert np.array_equal(np.isnan(g64[r]), np.isnan(g)), (r, np.isnan(g64[r]).nonzero()[0])
        if np.isnan(want):
            assert np.isnan(l64[r]) and np.isnan(g).all(), r
            continue
        bound = np.maximum(1.0, abs(w64[r])) * gerr
        off = abs(g64[r] - w64[r] * g)
        assert np.isfinite(bound).all() and (off <= bound).all(), (r, off.argmax(), off.max())
        # the loss is a 32-bit number: from 2^128 (1 - 2^-25) on the nearest is inf
        if abs(want) >= 2.0 ** 128 * (1 - 2.0 ** -25):
            want = np.copysign(INF, want)
        assert l64[r] == want or abs(l64[r] - want) <= lerr, (r, l64[r], want, lerr)


# a thread a row; one CTA and a cluster; a CTA that streams; teams of 4 and of 8 lanes
@pytest.mark.parametrize("rows,size", [(40, 21), (40, 32), (40, 500), (24, 40001), (700, 900),
                                       (160, 9001), (150, 40001), (9503, 241), (4803, 800)])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_every_entry_of_special_rows(vocab, rows, size, dtype):
    k, low = 12, torch.finfo(dtype).min
    x = logits(rows, size, dtype, 2)
    v, t, norm = teacher(x, k, F32, 3, 1.5, True)
    idx = t.long()
    listed = torch.zeros_like(x, dtype=torch.bool).scatter_(1, idx, True)
    x[0] = torch.where(listed[0], x[0], -INF)              # no mass off the list
    x[1] = torch.where(listed[1], x[1], low)               # the lowest value off it
    x[2] = torch.where(listed[2], -INF, x[2])              # none on the list: loss +inf
    x[3] = torch.where(listed[3], low, x[3])
    x[4] = torch.where(listed[4], x[4] + 200.0, x[4])      # the list far above the rest
    x[5] = torch.where(listed[5], x[5] - 200.0, x[5])      # and far below it
    x[6] = low
    x[7] = 0.0
    x[8, idx[8, 1:]] = -INF                                # but one of the listed
    x[9, ::2] = -INF
    x[9].scatter_(0, idx[9], 1.0)
    x[10] = -INF                                           # no loss
    x[11, 5] = float("nan")
    x[12, 7] = INF
    x[13, idx[13, 2]] = float("nan")
    x[14, idx[14, 0]] = INF
    x[15] = float("nan")
    t[15] = -1                                             # no entries: not looked at
    t[16, 3:] = -1
    t[17, 4] = t[17, 9]
    t[18, :] = t[18, 0]
    v[19, 5:] = -INF
    t[20, 2] = size
    t[21, 0], t[21, 5] = t[21, 5].clone(), t[21, 0].clone()
    w = torch.rand(rows, generator=torch.Generator("cuda").manual_seed(1), device="cuda") + 0.5
    w[22 % rows] = 0.0
    w[23 % rows] = -1.0
    at = torch.tensor([*range(15), *range(16, 24), rows - 1], device="cuda").unique()
    for n in (None, norm):
        kw = dict(teacher_log_norm=n, temperature=1.5)
        loss, grad = vocab.distill_loss_and_grad(x, v, t, row_weights=w, **kw)
        keep = at[(at != 22 % rows) & (at != 20)]
        check_every_entry(loss[keep], grad[keep], x[keep], v[keep], t[keep],
                          None if n is None else n[keep], 1.5, w[keep])
        assert loss[20].isnan() and grad[20].isnan().all()
        assert loss[15] == 0 and (grad[15] == 0).all() and (grad[22] == 0).all()
        z = x.clone().requires_grad_()
        l2 = vocab.distill_loss(z, v, t, **kw)
        (g2,) = torch.autograd.grad(l2, z, w)
        for a, b in ((l2.detach(), loss), (g2, grad)):
            assert torch.equal(a.isnan(), b.isnan())
            assert torch.equal(a.nan_to_num(-7.0), b.nan_to_num(-7.0))
