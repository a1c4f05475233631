"""Teacher numbers that are no numbers make their row's loss and gradient NaN, in
every kernel, and no other row's.  On a B200."""
import pytest
import torch

from test_gpu_vocab import logits, teacher

pytestmark = pytest.mark.gpu

INF, NAN = float("inf"), float("nan")
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


@pytest.fixture(scope="module")
def vocab():
    from hikoboshi_b200 import vocab
    return vocab


# a thread a row; one CTA and a cluster; a CTA that streams; teams of 4 and of 8 lanes
@pytest.mark.parametrize("rows,size", [(150, 21), (12, 32), (12, 500), (12, 40000), (700, 900),
                                       (9500, 100), (4800, 800)])
@pytest.mark.parametrize("tdtype", [F32, F16, BF16])
@pytest.mark.parametrize("k", [4, 15])
def test_infinite_and_nan_teachers(vocab, rows, size, tdtype, k):
    x = logits(rows, size, F32, size)
    v, t, norm = teacher(x, k, tdtype, 3, 1.5, True)
    good = vocab.distill_loss_and_grad(x, v, t, teacher_log_norm=norm, temperature=1.5)
    renormalised = vocab.distill_loss_and_grad(x, v, t, temperature=1.5)
    v[0, 0], v[1, k - 1], v[2, 1] = INF, INF, NAN       # bad entries
    v[3, 2], t[3, 2] = INF, -1                          # no entry: its value is not looked at
    norm[4], norm[5], norm[6] = INF, -INF, NAN
    norm[7], t[7] = INF, -1                             # no entries: nor is its log-norm
    norm[8], v[8] = NAN, -INF
    v[9], norm[9] = INF, INF                            # all of them
    w = torch.full((rows,), 0.5, device="cuda")
    w[10], v[10, 0] = 0.0, INF                          # weight 0: gradient 0
    for n in (norm, None):
        bad = [0, 1, 2, 9] + ([4, 5, 6] if n is not None else [])
        kw = dict(teacher_log_norm=n, temperature=1.5)
        loss, grad = vocab.distill_loss_and_grad(x, v, t, row_weights=w, **kw)
        assert loss[bad].isnan().all() and grad[bad].isnan().all()
        assert loss[10].isnan() and (grad[10] == 0).all()
        assert (loss[[7, 8]] == 0).all() and (grad[[7, 8]] == 0).all()
        fine = torch.ones(rows, dtype=torch.bool, device="cuda")
        fine[bad + [10]] = False
        assert loss[fine].isfinite().all() and grad[fine].isfinite().all()
        # the rows that nothing was done to are what they were
        same = list(range(11, rows)) + ([] if n is not None else [4, 5, 6])
        want = good if n is not None else renormalised
        assert torch.equal(loss[same], want[0][same])
        assert torch.equal(grad[same], want[1][same] * 0.5)
        z = x.clone().requires_grad_()
        l2 = vocab.distill_loss(z, v, t, **kw)
        (g2,) = torch.autograd.grad(l2, z, w)
        for a, b in ((l2.detach(), loss), (g2, grad)):
            assert torch.equal(a.isnan(), b.isnan())
            assert torch.equal(a.nan_to_num(-7.0), b.nan_to_num(-7.0))
