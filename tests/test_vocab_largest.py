"""The largest vocabulary that is accepted: slices of 128 KB, 17 steps a warp, the
longest map of marks, the longest listing.  On a B200.

The bounds of vocab_reference.sum_error count 160 additions one after another.
A thread that streams 512 of 262,144 tokens adds them 16 (8 of 32 bits) in turn to
a sum of their own and that sum to its running one, 16 (32) times; 9 joins of
threads follow, of 4 roundings each: 16 + 16 + 36 (8 + 32 + 36) and one rescaling
of 3 roundings for each new maximum.  In shared memory a thread adds 64."""
import pytest
import torch

from test_gpu_vocab import check_distill, check_sample, check_top, edge_rows, gen, logits, teacher

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
SIZE = 262144
FILTERS = [dict(), dict(top_k=50, top_p=0.95), dict(top_k=1024), dict(top_k=3000),
           dict(top_p=0.5), dict(top_p=0.97), dict(min_p=0.05), dict(temperature=0.0),
           dict(top_p=0.9, min_p=0.02, temperature=0.7), dict(top_p=0.99, temperature=3.0)]


@pytest.fixture(scope="module")
def vocab():
    from hikoboshi_b200 import vocab
    return vocab


def offset_rows(rows, dtype, seed, offset):
    base = logits(1, rows * (SIZE + 5) + 16, dtype, seed)[0]
    return base[offset:offset + rows * (SIZE + 5)].view(rows, SIZE + 5)[:, :SIZE]


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("rows", [1, 3, 40])
def test_largest_rows_held_by_a_cluster(vocab, rows, dtype):
    for offset in (0, 3):
        x = offset_rows(rows, dtype, rows + offset, offset)
        x[-1, -1] = 40.0 if dtype == F32 else 30.0  # the last token of the last slice
        at = torch.tensor([0, rows // 2, rows - 1], device="cuda").unique()
        for v in (0.0, 0.37, 1.0):
            u = torch.full((rows,), v, device="cuda")
            for f in FILTERS:
                got = vocab.sample_tokens(x, u, **f)
                check_sample([a[at] for a in got], x[at], u[at], **f)
        for k in (1, 64, 1024):
            check_top([a[at] for a in vocab.top_logits(x, k)], x[at], k)
        for k in (5, 1024):
            for tail in (False, True):
                v, t, norm = teacher(x, k, F32, k, 1.5, tail)
                kw = dict(teacher_log_norm=norm, temperature=1.5)
                loss, grad = vocab.distill_loss_and_grad(x, v, t, **kw)
                check_distill(loss[at], grad[at], x[at], v[at], t[at], norm[at] if tail else None,
                              1.5)
                z = x.detach().requires_grad_()
                l2 = vocab.distill_loss(z, v, t, **kw)
                (g2,) = torch.autograd.grad(l2.sum(), z)
                assert torch.equal(l2, loss) and torch.equal(g2, grad)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_largest_rows_streamed(vocab, dtype):
    rows = 600
    x = offset_rows(rows, dtype, 5, 1)
    x[-1, -1] = 30.0
    at = torch.tensor([0, 301, rows - 1], device="cuda")
    for k in (3, 1024):
        check_top([a[at] for a in vocab.top_logits(x, k, temperature=2.0)], x[at], k, 2.0)
    g = gen(1)
    t = torch.randint(0, SIZE, (rows, 1024), generator=g, device="cuda", dtype=torch.int32)
    t[:, :2] = torch.tensor([0, SIZE - 1], device="cuda", dtype=torch.int32)
    t[301, 7] = t[301, 9]
    v = torch.randn(rows, 1024, generator=g, device="cuda")
    norm = torch.full((rows,), 9.0, device="cuda")
    out = torch.empty_like(x)
    for n in (None, norm):
        kw = dict(teacher_log_norm=n, temperature=1.5)
        loss, grad = vocab.distill_loss_and_grad(x, v, t, grad_out=out, **kw)
        check_distill(loss[at], grad[at], x[at], v[at], t[at], None if n is None else n[at], 1.5)
        z = x.detach().requires_grad_()
        l2 = vocab.distill_loss(z, v, t, **kw)
        (g2,) = torch.autograd.grad(l2.sum(), z)
        assert torch.equal(l2, loss) and torch.equal(g2, grad)
        del z, l2, g2
    t[0, 5] = SIZE
    loss, grad = vocab.distill_loss_and_grad(x, v, t, grad_out=out)
    assert loss[0].isnan() and grad[0].isnan().all() and loss[1:].isfinite().all()


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_largest_rows_with_masks_and_equal_values(vocab, dtype):
    x = edge_rows(SIZE, dtype)
    u = torch.full((len(x),), 0.3, device="cuda")
    for f in FILTERS:
        check_sample(vocab.sample_tokens(x, u, **f), x, u, **f)
    for k in (1, 300):
        check_top(vocab.top_logits(x, k), x, k)
