"""The operators on vocabulary rows on a B200, against their definitions in 64
bits (tests/vocab_reference.py), at the sizes and masks where they can go wrong."""
import threading

import numpy as np
import pytest
import torch

from vocab_reference import distill_row, sample_row, to64, top_row

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
INF = float("inf")
TYPES = [F32, F16, BF16]
# one token, fewer than a warp, around its size, one and several CTAs a row
SIZES = [1, 2, 21, 31, 32, 33, 64, 257, 1000, 4097, 32768, 50001, 131072]


@pytest.fixture(scope="module")
def vocab():
    from hikoboshi_b200 import vocab
    return vocab


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def logits(rows, size, dtype, seed, scale=2.0):
    g = gen(seed)
    x = torch.randn(rows, size, generator=g, device="cuda") * scale
    x -= 0.7 * torch.rand(rows, size, generator=g, device="cuda").clamp(min=1e-7).log()
    return x.to(dtype)


def check_sample(got, x, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    x64, u64 = to64(x).reshape(-1, x.shape[-1]), to64(u).reshape(-1)
    n = len(u64)

    def per_row(v, cast):
        v = to64(v).reshape(-1) if isinstance(v, torch.Tensor) else np.full(n, cast(v))
        return v.astype(np.float64)

    t, k = per_row(temperature, np.float32), per_row(top_k, int)
    p, m = per_row(top_p, np.float32), per_row(min_p, np.float32)
    tokens, lps, kept = (a.cpu().numpy().reshape(-1) for a in got)
    for r in range(n):
        token, lp, count = sample_row(x64[r], u64[r], t[r], int(k[r]), p[r], m[r],
                                      drawn=int(tokens[r]))
        where = (r, x.shape, x.dtype, t[r], k[r], p[r], m[r], u64[r])
        assert tokens[r] == token and kept[r] == count, (tokens[r], token, kept[r], count, where)
        # one rounding of a 64-bit value
        if np.isfinite(lp):
            assert abs(lps[r] - lp) <= 2.0 ** -24 * abs(lp) + 1e-12, (lps[r], lp, where)
        else:
            assert np.array_equal(lps[r], np.float32(lp), equal_nan=True), (lps[r], lp, where)


def check_top(got, x, k, temperature=1.0):
    values, tokens, norm = got
    size = x.shape[-1]
    x2 = x.reshape(-1, size)
    x64 = to64(x2)
    v, t, nrm = (to64(values).reshape(-1, k), tokens.cpu().numpy().reshape(-1, k),
                 to64(norm).reshape(-1))
    for r in range(len(x64)):
        order, want, err = top_row(x64[r], k, float(np.float32(temperature)))
        assert np.array_equal(t[r], order), (r, t[r], order)
        taken = order >= 0
        assert np.array_equal(v[r][taken], x64[r][order[taken]]), r
        assert (v[r][~taken] == -INF).all()
        if np.isfinite(want):
            assert abs(nrm[r] - want) <= err, (r, nrm[r], want, err)
        else:
            assert nrm[r] == want, (r, nrm[r], want)


def teacher(x, k, dtype, seed, tau, tail):
    """A teacher near the student: listed values and tokens, log-norm or None."""
    a = x.float() + torch.randn(x.shape, generator=gen(seed), device="cuda")
    v, t = a.topk(k, dim=-1)
    norm = torch.logsumexp(a / tau, dim=-1) if tail else None
    return v.to(dtype).contiguous(), t.int().contiguous(), norm


def check_distill(loss, grad, x, values, tokens, norm, tau, weights=None):
    size = x.shape[-1]
    x64 = to64(x).reshape(-1, size)
    k = values.shape[-1]
    v64, t64 = to64(values).reshape(-1, k), tokens.cpu().numpy().reshape(-1, k)
    n64 = None if norm is None else to64(norm).reshape(-1)
    w64 = np.ones(len(x64)) if weights is None else to64(weights).reshape(-1)
    l64 = None if loss is None else to64(loss).reshape(-1)
    g64 = None if grad is None else to64(grad).reshape(-1, size)
    for r in range(len(x64)):
        want, g, lerr, gerr = distill_row(x64[r], v64[r], t64[r], None if n64 is None else n64[r],
                                          float(np.float32(tau)), x.dtype)
        if l64 is not None:
            if np.isfinite(want):
                assert abs(l64[r] - want) <= lerr, (r, l64[r], want, lerr)
            else:
                assert np.array_equal(l64[r], want, equal_nan=True), (r, l64[r], want)
        if g64 is not None:
            # the bound scales with the weight, but for the smallest numbers
            bound = np.maximum(1.0, abs(w64[r])) * gerr
            off = abs(g64[r] - w64[r] * g) - bound
            assert np.isnan(g).all() == np.isnan(g64[r]).all(), r
            assert not (off > 0).any(), (r, off.argmax(), g64[r][off.argmax()],
                                         w64[r] * g[off.argmax()], bound[off.argmax()])


# -- sampling -----------------------------------------------------------------

FILTERS = [dict(), dict(top_k=1), dict(top_k=7), dict(top_k=200, top_p=0.9), dict(top_p=0.5),
           dict(top_p=0.97), dict(min_p=0.05), dict(top_p=0.9, min_p=0.02, temperature=0.7),
           dict(top_k=40, top_p=0.95, min_p=0.01, temperature=1.3), dict(temperature=0.0),
           dict(top_p=0.0), dict(top_k=5000), dict(min_p=1.0)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("size", SIZES)
def test_sample_sizes_and_filters(vocab, size, dtype):
    rows = 3 if size > 5000 else 9
    for i, f in enumerate(FILTERS):
        x = logits(rows, size, dtype, 17 * size + i)
        u = torch.rand(rows, generator=gen(i), device="cuda")
        check_sample(vocab.sample_tokens(x, u, **f), x, u, **f)


@pytest.mark.parametrize("size", [21, 300, 40000])
def test_sample_settings_per_row(vocab, size):
    rows = 64
    x = logits(rows, size, BF16, size)
    g = gen(5)
    u = torch.rand(rows, generator=g, device="cuda", dtype=torch.float64)
    s = dict(temperature=torch.rand(rows, generator=g, device="cuda") * 1.5,
             top_k=torch.randint(0, 30, (rows,), generator=g, device="cuda", dtype=torch.int32),
             top_p=torch.rand(rows, generator=g, device="cuda"),
             min_p=torch.rand(rows, generator=g, device="cuda") * 0.1)
    s["temperature"][:5] = 0.0
    s["top_p"][5:9] = 1.0
    check_sample(vocab.sample_tokens(x, u, **s), x, u, **s)


def test_sample_row_settings_out_of_range_give_no_token(vocab):
    rows, size = 12, 100
    x = logits(rows, size, F32, 1)
    u = torch.full((rows,), 0.5, device="cuda")
    s = dict(temperature=torch.ones(rows, device="cuda"),
             top_k=torch.zeros(rows, dtype=torch.int32, device="cuda"),
             top_p=torch.ones(rows, device="cuda"), min_p=torch.zeros(rows, device="cuda"))
    s["temperature"][0], s["temperature"][1], s["temperature"][2] = -1.0, float("nan"), INF
    s["top_k"][3] = -1
    s["top_p"][4], s["top_p"][5], s["min_p"][6], s["min_p"][7] = 1.5, float("nan"), -0.1, 1.1
    u[8], u[9], u[10] = -0.1, float("nan"), 1.01
    for xx in (x, x[:, :21], x.repeat(1, 700)):
        got = vocab.sample_tokens(xx, u, **s)
        assert (got.tokens[:11] == -1).all() and (got.kept[:11] == 0).all()
        assert got.log_probs[:11].isnan().all() and got.tokens[11] >= 0
        check_sample(got, xx, u, **s)


def edge_rows(size, dtype):
    """Rows that masks, infinities and equal values make special."""
    low = torch.finfo(dtype).min
    x = logits(14, size, dtype, 3)
    x[0] = -INF                       # nothing left
    x[1] = low                        # masked with the type's lowest value
    x[2] = low
    x[2, size // 2] = 1.0
    x[3] = -INF
    x[3, -1] = -5.0                   # one token left, the last
    x[4, ::2] = -INF
    x[5] = 0.0                        # all equal
    x[6, 0] = INF
    x[6, -1] = INF
    x[7, : size // 2] = float("nan")
    x[8] = float("nan")
    x[9] = (x[9].float() * 2).round() / 2   # many equal values
    x[10] = 0.0
    x[10, ::3] = -0.0                 # both zeros are one value
    x[11] = low
    x[11, 0] = torch.finfo(dtype).max
    x[12] = -INF
    x[12, 0] = low
    x[13] = float("nan")
    x[13, size // 3] = -INF
    return x


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("size", [2, 21, 32, 100, 5000, 70001])
def test_sample_edges(vocab, size, dtype):
    x = edge_rows(size, dtype)
    for f in FILTERS:
        for v in (0.0, 0.3, 0.999999, 1.0):
            u = torch.full((len(x),), v, device="cuda")
            check_sample(vocab.sample_tokens(x, u, **f), x, u, **f)


@pytest.mark.parametrize("size", [21, 513, 60000])
def test_sample_flat_and_tied_rows(vocab, size):
    # equal weights are exact, so are their borders: half of the tokens, in index order
    x = torch.zeros(4, size, device="cuda")
    u = torch.tensor([0.0, 0.25, 0.5, 0.75], device="cuda")
    got = vocab.sample_tokens(x, u, top_p=0.5)
    n = -(-size // 2)
    assert (got.kept == n).all()
    assert got.tokens.tolist() == [int(v * n) for v in (0.0, 0.25, 0.5, 0.75)]
    flat = logits(4, size, F32, 9, scale=0.01) * 0.01
    for f in (dict(top_p=0.9), dict(top_k=size // 2), dict(top_k=size - 1, top_p=0.7)):
        check_sample(vocab.sample_tokens(flat, u, **f), flat, u, **f)


def test_sample_follows_the_distribution(vocab):
    # 60,000 draws from one row (row stride 0): a count is binomial, six sigma
    n = 60000
    x = logits(1, 21, F32, 4).expand(n, 21)
    u = torch.rand(n, generator=gen(8), device="cuda")
    p = torch.softmax(x[0].double(), 0).cpu().numpy()
    count = torch.bincount(vocab.sample_tokens(x, u).tokens.long(), minlength=21).cpu().numpy()
    assert (abs(count - n * p) <= 6 * np.sqrt(n * p * (1 - p)) + 1).all()


# -- the largest logits -------------------------------------------------------

@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("size", SIZES)
def test_top_sizes(vocab, size, dtype):
    rows = 3 if size > 5000 else 9
    for k in sorted({1, 2, 8, 33, 64, 256, 1024, min(size, 1024)}):
        x = logits(rows, size, dtype, size + k)
        for temperature in (1.0, 2.5):
            check_top(vocab.top_logits(x, k, temperature=temperature), x, k, temperature)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("size", [2, 21, 32, 100, 5000, 70001])
def test_top_edges(vocab, size, dtype):
    x = edge_rows(size, dtype)
    for k in (1, 5, 300):
        check_top(vocab.top_logits(x, k), x, k)


def test_top_of_sorted_rows(vocab):
    # all the large logits side by side, at either end
    for size in (3100, 100000):
        x = torch.arange(size, device="cuda", dtype=F32)[None] * 1e-3
        x = torch.cat([x, x.flip(1)])
        for k in (10, 1000):
            check_top(vocab.top_logits(x, k), x, k)


# -- distillation -------------------------------------------------------------

@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("size", SIZES)
def test_distill_sizes(vocab, size, dtype):
    rows = 3 if size > 5000 else 9
    for k in sorted({min(size, n) for n in (1, 5, 21, 64, 300)}):
        for tail in (False, True):
            for tau, tdtype in ((1.0, F32), (2.5, dtype)):
                x = logits(rows, size, dtype, size + k)
                v, t, norm = teacher(x, k, tdtype, k, tau, tail)
                w = torch.rand(rows, generator=gen(k), device="cuda") + 0.25
                w[0] = 0.0
                kw = dict(teacher_log_norm=norm, temperature=tau)
                loss, grad = vocab.distill_loss_and_grad(x, v, t, row_weights=w, **kw)
                check_distill(loss, grad, x, v, t, norm, tau, w)
                xr = x.clone().requires_grad_()
                l2 = vocab.distill_loss(xr, v, t, **kw)
                (g2,) = torch.autograd.grad(l2, xr, w)
                assert torch.equal(l2, loss) and torch.equal(g2, grad)


@pytest.mark.parametrize("size", [21, 500, 40000])
@pytest.mark.parametrize("tail", [False, True])
def test_distill_listings(vocab, size, tail):
    """Padding, tokens listed twice, entries of -inf, empty and bad listings."""
    rows, k = 8, 12
    x = logits(rows, size, F32, 2)
    v, t, norm = teacher(x, k, F32, 3, 1.0, True)
    t[0] = -1                                   # no entries
    t[1, 3:] = -1                               # padded
    t[2, 4] = t[2, 9]                           # the same token twice
    t[3, :] = t[3, 0]                           # always the same
    v[4, 5:] = -INF                             # masked entries
    v[5] = -INF                                 # none left
    t[6, 2] = size                              # out of the vocabulary
    x[0] = float("nan")                         # not looked at: the row has no entries
    x[7, t[7, 1].long()] = -INF                 # a listed token the student masks out
    norm = norm if tail else None
    loss, grad = vocab.distill_loss_and_grad(x, v, t, teacher_log_norm=norm)
    assert loss[0] == 0 and (grad[0] == 0).all() and loss[5] == 0 and (grad[5] == 0).all()
    assert loss[6].isnan() and grad[6].isnan().all() and loss[7] == INF
    x[0] = 0
    check_distill(loss, grad, x, v, t, norm, 1.0)
    w = torch.zeros(rows, device="cuda")
    x[0] = float("nan")
    loss, grad = vocab.distill_loss_and_grad(x, v, t, teacher_log_norm=norm, row_weights=w)
    assert (grad == 0).all()


@pytest.mark.parametrize("size", [21, 700, 33333])
def test_distill_student_rows_without_a_loss_are_nan(vocab, size):
    x = logits(4, size, F32, 2)
    v, t, norm = teacher(x, 3, F32, 3, 1.0, True)
    x[0] = -INF
    x[1, 5] = float("nan")
    x[2, 7] = INF
    for n in (None, norm):
        loss, grad = vocab.distill_loss_and_grad(x, v, t, teacher_log_norm=n)
        assert loss[:3].isnan().all() and grad[:3].isnan().all()
        check_distill(loss[3:], grad[3:], x[3:], v[3:], t[3:], n[3:] if n is not None else None, 1.0)


@pytest.mark.parametrize("dtype", TYPES)
def test_distill_masked_student(vocab, dtype):
    for size in (21, 900, 50001):
        x = logits(3, size, dtype, 6)
        v, t, norm = teacher(x, 4, F32, 3, 1.0, True)
        keep = torch.zeros_like(x, dtype=torch.bool).scatter_(1, t.long(), True)
        x[0] = torch.where(keep[0], x[0], -INF)                       # no mass off the list
        x[1] = torch.where(keep[1], x[1], torch.finfo(dtype).min)     # the lowest value
        loss, grad = vocab.distill_loss_and_grad(x[:1], v[:1], t[:1], teacher_log_norm=norm[:1])
        check_distill(loss, grad, x[:1], v[:1], t[:1], norm[:1], 1.0)
        assert (grad[0][~keep[0]] == 0).all()
        loss, grad = vocab.distill_loss_and_grad(x, v, t)
        check_distill(loss, grad, x, v, t, None, 1.0)


@pytest.mark.parametrize("size", [21, 400, 20000])
@pytest.mark.parametrize("tail", [False, True])
def test_distill_gradient_against_differences(vocab, size, tail):
    # along v in {-1, 0, 1}^V: the third derivative of the loss is at most
    # tau^2 * 2 * (2 / tau)^3, the loss is off by its bound on both sides
    tau, h = 1.5, 2.0 ** -5
    x = (logits(4, size, F32, 1) * 1024).round() / 1024
    v, t, norm = teacher(x, 6, F32, 3, tau, tail)
    d = torch.randint(-1, 2, x.shape, generator=gen(4), device="cuda").float()
    kw = dict(teacher_log_norm=norm, temperature=tau)
    up, down = vocab.distill_loss(x + h * d, v, t, **kw), vocab.distill_loss(x - h * d, v, t, **kw)
    _, grad = vocab.distill_loss_and_grad(x, v, t, **kw)
    slope = (grad.double() * d).sum(1).cpu().numpy()
    diff = ((up.double() - down.double()) / (2 * h)).cpu().numpy()
    for r in range(4):
        errs = [distill_row(to64(y[r]), to64(v[r]), t[r].cpu().numpy(),
                            None if norm is None else float(norm[r]), tau, F32)
                for y in (x + h * d, x - h * d, x)]
        bound = (errs[0][2] + errs[1][2]) / (2 * h) + errs[2][3].sum()
        bound += h * h / 6 * tau * tau * 2 * (2 / tau) ** 3
        assert abs(slope[r] - diff[r]) <= bound, (slope[r], diff[r], bound)


# -- layouts, streams, graphs -------------------------------------------------

@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("size", [21, 1001, 45000])
def test_views_at_any_offset_and_stride(vocab, size, dtype):
    rows, k = 5, 9
    base = logits(1, rows * (size + 13) + 16, dtype, 5)[0]
    for offset in range(8):
        x = base[offset:offset + rows * (size + 13)].view(rows, size + 13)[:, :size]
        u = torch.rand(rows, generator=gen(offset), device="cuda")
        check_sample(vocab.sample_tokens(x, u, top_p=0.9), x, u, top_p=0.9)
        check_top(vocab.top_logits(x, k), x, k)
        v, t, norm = teacher(x, k, F32, 3, 1.0, True)
        # the gradient goes between guard values, at another offset
        out = torch.full((rows * (size + 5) + 16,), 7.0, dtype=dtype, device="cuda")
        at = (3 * offset) % 8
        g = out[at:at + rows * (size + 5)].view(rows, size + 5)[:, :size]
        loss, grad = vocab.distill_loss_and_grad(x, v, t, teacher_log_norm=norm, grad_out=g)
        check_distill(loss, grad, x, v, t, norm, 1.0)
        g.fill_(7.0)
        assert (out == 7.0).all()


def test_leading_dimensions_and_one_row(vocab):
    x = logits(6, 21, F32, 1).view(2, 3, 21)
    u = torch.rand(2, 3, generator=gen(1), device="cuda")
    got = vocab.sample_tokens(x, u, top_k=4)
    assert got.tokens.shape == (2, 3)
    check_sample(got, x, u, top_k=4)
    top = vocab.top_logits(x, 4)
    assert top.values.shape == (2, 3, 4)
    check_top(top, x, 4)
    loss, grad = vocab.distill_loss_and_grad(x, top.values, top.tokens,
                                             teacher_log_norm=top.log_norm)
    assert loss.shape == (2, 3) and grad.shape == x.shape
    # a student that is its teacher: no loss (its bound aside)
    check_distill(loss, grad, x, top.values, top.tokens, top.log_norm, 1.0)
    one = x[0, 0]
    got = vocab.sample_tokens(one, u[0, 0], top_p=0.5)
    assert got.tokens.shape == ()
    check_sample(got, one, u[0, 0], top_p=0.5)
    loss, grad = vocab.distill_loss_and_grad(one, top.values[0, 0], top.tokens[0, 0])
    assert loss.shape == () and grad.shape == (21,)


@pytest.mark.parametrize("size", [21, 999, 64000])
@pytest.mark.parametrize("dtype", TYPES)
def test_gradient_in_place_of_the_logits(vocab, size, dtype):
    x = logits(7, size, dtype, 1)
    v, t, norm = teacher(x, 5, F32, 3, 1.0, True)
    loss, grad = vocab.distill_loss_and_grad(x, v, t, teacher_log_norm=norm)
    y = x.clone()
    loss2, grad2 = vocab.distill_loss_and_grad(y, v, t, teacher_log_norm=norm, grad_out=y)
    assert grad2.data_ptr() == y.data_ptr()
    assert torch.equal(loss, loss2) and torch.equal(grad, y)


def test_gradient_in_place_counts_as_a_change(vocab):
    x = logits(7, 50, F32, 1)
    v, t, _ = teacher(x, 5, F32, 3, 1.0, False)
    x.requires_grad_()
    y = x * 1.0
    square = (y * y).sum()  # its backward pass needs y
    before = y._version
    vocab.distill_loss_and_grad(y.detach(), v, t, grad_out=y.detach())
    assert y._version > before
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        square.backward()


@pytest.mark.parametrize("size", [21, 5000])
def test_broadcast_weights_and_shared_rows(vocab, size):
    x = logits(1, size, F32, 1)
    v, t, _ = teacher(x.expand(6, size), 5, F32, 3, 1.0, False)
    leaf = x.clone().requires_grad_()
    vocab.distill_loss(leaf.expand(6, size), v, t).sum().backward()   # weights of stride 0
    _, each = vocab.distill_loss_and_grad(x.expand(6, size), v, t)
    # six f32 numbers added: five roundings of at most their absolute sum
    bound = 5 * 2.0 ** -24 * each.abs().sum(0)
    assert ((leaf.grad[0].double() - each.double().sum(0)).abs() <= bound).all()
    w = torch.arange(12, device="cuda", dtype=F32)[::2]
    _, g = vocab.distill_loss_and_grad(x.expand(6, size), v, t, row_weights=w)
    check_distill(None, g, x.expand(6, size), v, t, None, 1.0, w)


def test_offsets_past_32_bits(vocab):
    # the second row starts 2^31 + 5 elements behind the first
    size, stride = 2000, 2 ** 31 + 5
    buf = torch.zeros(stride + size, dtype=BF16, device="cuda")
    x = buf.as_strided((2, size), (stride, 1))
    x.copy_(logits(2, size, BF16, 1))
    u = torch.tensor([0.2, 0.7], device="cuda")
    check_sample(vocab.sample_tokens(x, u, top_p=0.9), x, u, top_p=0.9)
    check_top(vocab.top_logits(x, 20), x, 20)
    v, t, norm = teacher(x, 20, F32, 3, 1.0, True)
    want = vocab.distill_loss_and_grad(x.contiguous(), v, t, teacher_log_norm=norm)
    got = vocab.distill_loss_and_grad(x, v, t, teacher_log_norm=norm, grad_out=x)
    assert torch.equal(want[0], got[0]) and torch.equal(want[1], x)


def test_rows_behind_the_last_are_left_alone(vocab):
    for size in (21, 2900):
        buf = logits(10, size, F32, 1)
        guard = buf[6:].clone()
        x = buf[:6]
        v, t, norm = teacher(x, 4, F32, 1, 1.0, True)
        vocab.distill_loss_and_grad(x, v, t, teacher_log_norm=norm, grad_out=x)
        assert torch.equal(buf[6:], guard)


def run_all(vocab, x, u, w):
    s = vocab.sample_tokens(x, u, temperature=0.8, top_p=0.95, min_p=0.01)
    top = vocab.top_logits(x, 16, temperature=2.0)
    student = (x.float() * 0.7).to(x.dtype)
    loss, grad = vocab.distill_loss_and_grad(student, top.values, top.tokens, row_weights=w,
                                             teacher_log_norm=top.log_norm, temperature=2.0)
    return (*s, *top, loss, grad)


@pytest.mark.parametrize("size,rows", [(21, 2900), (1500, 40), (80000, 6)])
def test_a_run_repeats_bit_for_bit_on_other_streams_and_in_graphs(vocab, size, rows):
    x = logits(rows, size, BF16, 1)
    u = torch.rand(rows, generator=gen(2), device="cuda")
    w = torch.rand(rows, generator=gen(3), device="cuda")
    want = run_all(vocab, x, u, w)
    check_sample([a[:6] for a in want[:3]], x[:6], u[:6], temperature=0.8, top_p=0.95, min_p=0.01)
    check_top([a[:8] for a in want[3:6]], x[:8], 16, 2.0)
    check_distill(want[6][:8], want[7][:8], (x.float() * 0.7).to(BF16)[:8], want[3][:8],
                  want[4][:8], want[5][:8], 2.0, w[:8])
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = []
    for st in streams:
        with torch.cuda.stream(st):
            got.append(run_all(vocab, x, u, w))
    torch.cuda.synchronize()
    for g in got:
        assert all(torch.equal(a, b) for a, b in zip(g, want))
    graphs, outs = [], []
    xs = [x.clone(), logits(rows, size, BF16, 7)]
    for y in xs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(run_all(vocab, y, u, w))
        graphs.append(g)
    want2 = run_all(vocab, xs[1], u, w)
    torch.cuda.synchronize()
    for st, g in zip(streams, graphs):
        with torch.cuda.stream(st):
            for _ in range(3):
                g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(outs[0], want))
    assert all(torch.equal(a, b) for a, b in zip(outs[1], want2))
    xs[0].copy_(xs[1])       # new inputs, same graph: nothing is kept from the capture
    graphs[0].replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(outs[0], want2))


def test_two_threads_at_once(vocab):
    inputs = [logits(200, 5000, F32, s) for s in range(2)]
    u = torch.rand(200, generator=gen(2), device="cuda")
    want = [run_all(vocab, x, u, u) for x in inputs]
    torch.cuda.synchronize()
    bad = []

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                got = run_all(vocab, inputs[i], u, u)
            torch.cuda.current_stream().synchronize()
            bad.extend(not torch.equal(a, b) for a, b in zip(got, want[i]))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert len(bad) == 16 and not any(bad)


def test_autograd_is_refused_in_a_capture(vocab):
    from hikoboshi_b200 import HkbError
    x = logits(4, 50, F32, 1).requires_grad_()
    v, t, _ = teacher(x.detach(), 3, F32, 1, 1.0, False)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        with pytest.raises(HkbError) as e:
            vocab.distill_loss(x, v, t)
        out = vocab.distill_loss(x.detach(), v, t)
    assert e.value.code == 2
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, vocab.distill_loss(x.detach(), v, t))


def test_gpu_refusals(vocab):
    from hikoboshi_b200 import HkbError
    x, u = logits(3, 21, F32, 1), torch.zeros(3)
    for call in (lambda: vocab.sample_tokens(x, u),
                 lambda: vocab.sample_tokens(x.cpu(), u),
                 lambda: vocab.sample_tokens(x, u.cuda(), top_p=torch.ones(3))):
        with pytest.raises(HkbError) as e:
            call()
        assert e.value.code == 1 and "device" in e.value.detail


# -- many rows: the kernels that stream rows instead of holding them ----------

MANY = 160


def pick(rows):
    """Rows that are compared: from the first CTAs, the last ones, and between."""
    return torch.tensor([0, 1, 2, 77, rows - 2, rows - 1], device="cuda")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("size", [33, 40, 257, 1001, 4097, 33003])
def test_many_rows_sizes(vocab, size, dtype):
    at = pick(MANY)
    x = logits(MANY, size, dtype, size)
    u = torch.rand(MANY, generator=gen(1), device="cuda")
    for f in FILTERS:
        got = vocab.sample_tokens(x, u, **f)
        check_sample([a[at] for a in got], x[at], u[at], **f)
    for k in (1, 8, 200, 1024):
        got = vocab.top_logits(x, k, temperature=0.7)
        check_top([a[at] for a in got], x[at], k, 0.7)
    for k in sorted({min(size, n) for n in (1, 40, 700)}):
        for tail in (False, True):
            v, t, norm = teacher(x, k, F32, k, 1.5, tail)
            w = torch.rand(MANY, generator=gen(k), device="cuda") + 0.25
            w[1] = 0.0
            loss, grad = vocab.distill_loss_and_grad(x, v, t, row_weights=w, temperature=1.5,
                                                     teacher_log_norm=norm)
            n = norm[at] if tail else None
            check_distill(loss[at], grad[at], x[at], v[at], t[at], n, 1.5, w[at])
            only = vocab.distill_loss(x, v, t, temperature=1.5, teacher_log_norm=norm)
            assert torch.equal(only, loss)
            y = x.clone()
            _, g2 = vocab.distill_loss_and_grad(y, v, t, row_weights=w, temperature=1.5,
                                                teacher_log_norm=norm, grad_out=y)
            assert torch.equal(g2, grad) and g2.data_ptr() == y.data_ptr()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("size", [33, 100, 5000, 20001])
def test_many_rows_edges(vocab, size, dtype):
    x = edge_rows(size, dtype).repeat(11, 1)
    n = len(x) // 11
    for k in (1, 5, 300, 1024):
        got = vocab.top_logits(x, k)
        check_top([a[:n] for a in got], x[:n], k)
        check_top([a[-n:] for a in got], x[-n:], k)
    for f in FILTERS:
        for v in (0.0, 0.3, 1.0):
            u = torch.full((len(x),), v, device="cuda")
            got = vocab.sample_tokens(x, u, **f)
            check_sample([a[-n:] for a in got], x[-n:], u[-n:], **f)
    # equal logits by the thousand: the list of candidates cannot hold them
    flat = torch.zeros(MANY, size, dtype=dtype, device="cuda")
    flat[:, size // 2] = 1.0
    check_top([a[:2] for a in vocab.top_logits(flat, 20)], flat[:2], 20)


@pytest.mark.parametrize("size", [50, 700, 9001])
@pytest.mark.parametrize("tail", [False, True])
def test_many_rows_listings(vocab, size, tail):
    k = 12
    x = logits(MANY, size, F32, 2)
    v, t, norm = teacher(x, k, F32, 3, 1.0, True)
    t[0] = -1
    t[1, 3:] = -1
    t[2, 4] = t[2, 9]
    t[3, :] = t[3, 0]
    v[4, 5:] = -INF
    v[5] = -INF
    t[6, 2] = size
    x[0] = float("nan")
    x[7, t[7, 1].long()] = -INF
    x[8] = -INF
    x[9, 5] = float("nan")
    x[10, 7] = INF
    x[11] = torch.finfo(F32).min
    v[12, 3] = float("nan")
    norm = norm if tail else None
    loss, grad = vocab.distill_loss_and_grad(x, v, t, teacher_log_norm=norm)
    assert loss[0] == 0 and (grad[0] == 0).all() and loss[5] == 0 and (grad[5] == 0).all()
    assert loss[7] == INF
    for r in (6, 8, 9, 10, 12):
        assert loss[r].isnan() and grad[r].isnan().all(), r
    x[0] = 0
    at = torch.tensor([0, 1, 2, 3, 4, 5, 6, 7, 11, 13, MANY - 1], device="cuda")
    check_distill(loss[at], grad[at], x[at], v[at], t[at], None if norm is None else norm[at], 1.0)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("size", [35, 1001, 9000])
def test_many_rows_at_any_offset_and_stride(vocab, size, dtype):
    base = logits(1, MANY * (size + 13) + 16, dtype, 5)[0]
    at = pick(MANY)
    for offset in range(8):
        x = base[offset:offset + MANY * (size + 13)].view(MANY, size + 13)[:, :size]
        check_top([a[at] for a in vocab.top_logits(x, 9)], x[at], 9)
        v, t, norm = teacher(x, 9, F32, 3, 1.0, True)
        out = torch.full((MANY * (size + 5) + 16,), 7.0, dtype=dtype, device="cuda")
        o = (3 * offset) % 8
        g = out[o:o + MANY * (size + 5)].view(MANY, size + 5)[:, :size]
        loss, grad = vocab.distill_loss_and_grad(x, v, t, teacher_log_norm=norm, grad_out=g)
        check_distill(loss[at], grad[at], x[at], v[at], t[at], norm[at], 1.0)
        g.fill_(7.0)
        assert (out == 7.0).all()


@pytest.mark.parametrize("size", [3, 8, 9, 21, 24, 25, 32, 60, 96, 97, 224, 225, 480, 481, 992, 993])
def test_near_ties_and_near_borders(vocab, size):
    # neighbours in the type: their order needs every bit, their sums borders
    # that 32 bits cannot tell apart
    rows = 200
    g = gen(size)
    step = torch.randint(0, 40, (rows, size), generator=g, device="cuda")
    x = (torch.full((rows, size), 1.0, device="cuda").view(torch.int32) + step.int()).view(F32)
    x[: rows // 2] = torch.where(step[: rows // 2] % 2 == 0, x[: rows // 2], -x[: rows // 2])
    u = torch.rand(rows, generator=g, device="cuda", dtype=torch.float64)
    for k in (1, 5, 16, 17, 40, size):
        check_top(vocab.top_logits(x, k), x, k)
    for f in (dict(top_k=5), dict(top_p=0.5), dict(top_k=7, top_p=0.6), dict(top_p=0.9, min_p=0.9),
              dict(top_k=max(1, size // 2))):
        check_sample(vocab.sample_tokens(x, u, **f), x, u, **f)
    # borders that lie exactly between two tokens, and a hair beside
    flat = torch.zeros(3, size, device="cuda")
    for n in {1, size // 2, size}:
        for p in (n / size, np.nextafter(np.float32(n / size), np.float32(2)),
                  np.nextafter(np.float32(n / size), np.float32(0))):
            p = float(min(1.0, p))
            v = torch.tensor([0.0, 0.5, 0.999], device="cuda")
            got = vocab.sample_tokens(flat, v, top_p=p)
            # p is a 32-bit number: the head is the least n with n / size >= p
            want = size if p == 1.0 else max(1, int(np.ceil(np.float64(np.float32(p)) * size)))
            assert (got.kept == want).all(), (size, p, got.kept, want)


def test_extreme_temperatures(vocab):
    for size in (21, 300, 5000, 70000):
        x = logits(4, size, F32, 1)
        x[1] *= 1e30
        x[2] = torch.finfo(F32).min
        x[2, 3] = torch.finfo(F32).max
        x[3] *= 1e-38
        u = torch.tensor([0.1, 0.5, 0.7, 0.9], device="cuda")
        for t in (1e-45, 1e-38, 1e-20, 1e20, 1e30, 3e38):
            for f in (dict(), dict(top_p=0.7), dict(top_k=5), dict(min_p=0.5), dict(top_p=0.3, top_k=9)):
                check_sample(vocab.sample_tokens(x, u, temperature=t, **f), x, u, temperature=t, **f)


@pytest.mark.parametrize("size", [2500, 60000])
def test_sampling_repeats_bit_for_bit_at_exact_borders(vocab, size):
    # rows that repeat themselves put borders exactly on u and p: whichever side
    # they fall, they fall the same way every time
    block = logits(1, size // 50, F32, 5)
    x = block.repeat(1, 50).expand(8, size).contiguous()
    x[4:] = (x[4:] * 4).round() / 4
    u = torch.tensor([0.1, 0.25, 0.5, 0.98] * 2, device="cuda")
    for f in (dict(), dict(top_p=0.5), dict(top_p=0.25, top_k=1000), dict(top_k=900),
              dict(top_p=0.75, temperature=2.0)):
        want = vocab.sample_tokens(x, u, **f)
        for _ in range(10):
            got = vocab.sample_tokens(x, u, **f)
            assert all(torch.equal(a, b) for a, b in zip(got, want)), f


def test_loss_is_differentiable_once(vocab):
    x = logits(4, 50, F32, 1).requires_grad_()
    v, t, _ = teacher(x.detach(), 3, F32, 1, 1.0, False)
    with pytest.raises(RuntimeError, match="differentiable once"):
        torch.autograd.grad(vocab.distill_loss(x, v, t).sum(), x, create_graph=True)


def test_extreme_distill_temperatures(vocab):
    for size in (21, 500, 30000):
        for rows in (3, 160):
            x = logits(rows, size, F32, 1)
            for tau in (1e-3, 1e4):
                v, t, norm = teacher(x, 5, F32, 2, tau, True)
                for n in (None, norm):
                    loss, grad = vocab.distill_loss_and_grad(x, v, t, teacher_log_norm=n,
                                                             temperature=tau)
                    check_distill(loss[:3], grad[:3], x[:3], v[:3], t[:3],
                                  None if n is None else n[:3], tau)
                check_top([a[:3] for a in vocab.top_logits(x, 5, temperature=tau)], x[:3], 5, tau)


@pytest.mark.parametrize("rows,size", [(5, 33), (5, 3001), (3, 70001), (160, 40), (160, 5003),
                                       (150, 40000), (2000, 700)])
@pytest.mark.parametrize("dtype", TYPES)
def test_backward_is_the_fused_gradient(vocab, rows, size, dtype):
    # to the bit, with every special row and from any offset
    base = logits(1, rows * (size + 3) + 16, dtype, 5)[0]
    for offset in (0, 3):
        x = base[offset:offset + rows * (size + 3)].view(rows, size + 3)[:, :size].clone() \
            if offset == 0 else base[offset:offset + rows * (size + 3)].view(rows, size + 3)[:, :size]
        v, t, norm = teacher(x, 20, dtype, 3, 1.5, True)
        w = torch.rand(rows, generator=gen(1), device="cuda") + 0.5
        w[2] = 0.0
        t[0] = -1
        t[1, 4] = t[1, 9]
        t[3 % rows, 2] = size if rows > 4 else t[3 % rows, 2]
        for n in (None, norm):
            kw = dict(teacher_log_norm=n, temperature=1.5)
            loss, grad = vocab.distill_loss_and_grad(x, v, t, row_weights=w, **kw)
            xr = x.detach().requires_grad_()
            l2 = vocab.distill_loss(xr, v, t, **kw)
            (g2,) = torch.autograd.grad(l2, xr, w)
            assert torch.equal(l2.nan_to_num(-7.0), loss.nan_to_num(-7.0))
            assert torch.equal(g2.nan_to_num(-7.0), grad.nan_to_num(-7.0))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("size", [225, 480, 481, 700, 992, 993, 5000])
def test_thousand_rows(vocab, size, dtype):
    edges = edge_rows(size, dtype)
    n = len(edges)
    x = torch.cat([logits(1100, size, dtype, size), edges])
    at = torch.cat([torch.arange(4), torch.arange(1100 - 3, 1100 + n)]).cuda()
    for f in FILTERS:
        for v in (0.0, 0.3, 1.0):
            u = torch.full((len(x),), v, device="cuda")
            got = vocab.sample_tokens(x, u, **f)
            check_sample([a[at] for a in got], x[at], u[at], **f)
    for k in (1, 8, 100, min(size, 1024)):
        got = vocab.top_logits(x, k)
        check_top([a[at] for a in got], x[at], k)
    y = x[:1100]
    for tail in (False, True):
        v, t, norm = teacher(y, 40, F32, 3, 1.5, tail)
        loss, grad = vocab.distill_loss_and_grad(y, v, t, temperature=1.5, teacher_log_norm=norm)
        assert torch.equal(vocab.distill_loss(y, v, t, temperature=1.5, teacher_log_norm=norm), loss)
        few = at[:7]
        check_distill(loss[few], grad[few], y[few], v[few], t[few],
                      norm[few] if tail else None, 1.5)


@pytest.mark.parametrize("size", [40, 225, 481, 992])
def test_thousand_rows_near_borders(vocab, size):
    # borders that 32 bits cannot place: neighbours in the type, a tail of
    # weights below the sums' rounding, differences that overflow 32 bits
    rows = 1100
    g = gen(size)
    step = torch.randint(0, 40, (rows, size), generator=g, device="cuda")
    near = (torch.full((rows, size), 1.0, device="cuda").view(torch.int32) + step.int()).view(F32)
    tail = -40.0 * torch.rand(rows, size, generator=g, device="cuda")
    huge = torch.finfo(F32).max * (2 * torch.rand(rows, size, generator=g, device="cuda") - 1)
    u = torch.rand(rows, generator=g, device="cuda", dtype=torch.float64)
    at = torch.arange(0, rows, 41, device="cuda")
    below = float(np.nextafter(np.float32(1), np.float32(0)))
    for x, temperature in ((near, 1.0), (tail, 1.0), (huge, 2e38)):
        for f in (dict(top_p=0.5), dict(top_p=0.9), dict(top_p=below),
                  dict(top_k=size // 2, top_p=0.9)):
            got = vocab.sample_tokens(x, u, temperature=temperature, **f)
            check_sample([a[at] for a in got], x[at], u[at], temperature=temperature, **f)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("size,offset", [(33, 0), (33, 1), (40, 3), (96, 0), (241, 5), (300, 0), (512, 1), (600, 1),
                                         (992, 0)])
def test_distill_thousands_of_short_rows(vocab, size, offset, dtype):
    # several rows to a warp; the last CTA is not full
    rows, k = 9503, 12
    pitch = size + 2 * offset
    base = logits(1, rows * pitch + offset, dtype, 2)[0]
    x = base[offset:].view(rows, pitch)[:, :size]
    v, t, norm = teacher(x, k, F32, 3, 1.5, True)
    t[0] = -1
    t[1, 3:] = -1
    t[2, 4] = t[2, 9]
    t[3, :] = t[3, 0]
    v[4, 5:] = -INF
    v[5] = -INF
    t[6, 2] = size
    x[0] = float("nan")
    x[7, t[7, 1].long()] = -INF
    x[8] = -INF
    x[9, 5] = float("nan")
    x[10, 7] = INF
    x[11] = torch.finfo(dtype).min
    v[12, 3] = float("nan")
    w = torch.rand(rows, generator=gen(1), device="cuda") + 0.5
    w[14] = 0.0
    at = torch.tensor([1, 2, 3, 4, 11, 13, 14, 15, 77, rows - 2, rows - 1], device="cuda")
    for n in (None, norm):
        kw = dict(teacher_log_norm=n, temperature=1.5)
        loss, grad = vocab.distill_loss_and_grad(x, v, t, row_weights=w, **kw)
        assert loss[0] == 0 and (grad[0] == 0).all() and loss[5] == 0 and (grad[5] == 0).all()
        assert loss[7] == INF and (grad[14] == 0).all()
        for r in (6, 8, 9, 10, 12):
            assert loss[r].isnan() and grad[r].isnan().all(), r
        check_distill(loss[at], grad[at], x[at], v[at], t[at], None if n is None else n[at], 1.5,
                      w[at])
        again = vocab.distill_loss(x, v, t, **kw)
        assert torch.equal(again.nan_to_num(-7.0), loss.nan_to_num(-7.0))
        # in place, and through autograd
        other = base.clone()
        y = other[offset:].view(rows, pitch)[:, :size]
        vocab.distill_loss_and_grad(y, v, t, row_weights=w, grad_out=y, **kw)
        assert torch.equal(y.nan_to_num(-7.0), grad.nan_to_num(-7.0))
        if offset:  # what lies between the rows stays
            assert torch.equal(other[offset:].view(rows, pitch)[:, size:],
                               base[offset:].view(rows, pitch)[:, size:])
        z = x.detach().requires_grad_()
        (g2,) = torch.autograd.grad(vocab.distill_loss(z, v, t, **kw), z, w)
        assert torch.equal(g2.nan_to_num(-7.0), grad.nan_to_num(-7.0))
    # from the shortest listing to the longest
    for n in sorted({1, 17, 33, min(size, 128), size}):
        v, t, norm = teacher(x[16:], n, F32, 5, 1.0, True)
        loss, grad = vocab.distill_loss_and_grad(x[16:], v, t, teacher_log_norm=norm)
        few = torch.tensor([0, 1, 2, rows - 18, rows - 17], device="cuda")
        check_distill(loss[few], grad[few], x[16:][few], v[few], t[few], norm[few], 1.0)


@pytest.mark.parametrize("size", [1500, 4000, 131072])
def test_sample_from_long_lists_of_neighbours(vocab, size):
    # heads of 193 to 2048 tokens whose indices lie close together, next to one far off
    g = gen(size)
    rows = 6
    x = torch.full((rows, size), -60.0, device="cuda")
    for r, (lo, n) in enumerate(((0, 300), (700, 500), (size - 260, 260), (5, 200), (100, 1200),
                                 (250, 400))):
        n = min(n, size - lo)
        x[r, lo:lo + n] = torch.rand(n, generator=g, device="cuda")
    x[3, size - 1] = 0.5
    x[5, 250:650] = 0.25  # equal logits
    for u in (0.0, 0.1, 0.5, 0.93, 1.0):
        us = torch.full((rows,), u, device="cuda", dtype=torch.float64)
        for f in (dict(top_p=0.9), dict(top_p=0.999), dict(top_k=250), dict(top_k=1000, top_p=0.95),
                  dict(top_p=0.97, min_p=0.5)):
            got = vocab.sample_tokens(x, us, **f)
            check_sample(got, x, us, **f)
            again = vocab.sample_tokens(x, us, **f)
            assert all(torch.equal(p, q) for p, q in zip(got, again))
