"""Sampling where 32 bits do not reach: temperatures whose reciprocal overflows
them, and the smallest uniforms.  On a B200, against the 64-bit definition."""
import pytest
import torch

from test_gpu_vocab import check_sample, gen, logits

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


@pytest.fixture(scope="module")
def vocab():
    from hikoboshi_b200 import vocab
    return vocab


# a thread, a warp and a CTA a row
@pytest.mark.parametrize("size,rows", [(2, 7), (21, 7), (32, 7), (33, 7), (100, 7), (224, 7),
                                       (900, 600), (900, 7), (5000, 7)])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_temperatures_below_the_smallest_normal_number(vocab, size, rows, dtype):
    x = logits(rows, size, dtype, size)
    x[1] = 0.0                              # all equal: top-p cuts by number
    x[2] = x[2].max()
    x[2, : size // 3] -= 1.0                # equal largest logits, not the first ones
    x[3] = torch.finfo(dtype).min
    x[3, size // 2] = torch.finfo(dtype).max
    x[4] = 0.0
    x[4, ::2] = 2.0 ** -149 if dtype == F32 else torch.finfo(dtype).smallest_normal
    steps = torch.randint(0, 4, (size,), generator=gen(1), device="cuda")
    x[5] = (steps.double() * 2.0 ** -149).to(dtype)  # logits as close as the temperature
    at = torch.arange(7, device="cuda")
    for t in (2.0 ** -149, 1e-44, 1e-40, 4.2e-39, 4.3e-39, 1e-38):
        for f in (dict(top_p=0.9), dict(top_p=0.5, top_k=max(1, size // 2)), dict(top_p=0.0),
                  dict(top_p=0.7, min_p=0.1), dict(top_k=3), dict()):
            for v in (0.0, 0.4, 0.9):
                u = torch.full((rows,), v, device="cuda")
                got = vocab.sample_tokens(x, u, temperature=t, **f)
                check_sample([a[at] for a in got], x[at], u[at], temperature=t, **f)


# a thread, a warp, a CTA and a cluster a row; lists of up to 192 tokens and longer ones
@pytest.mark.parametrize("size", [21, 200, 900, 5000, 60000])
@pytest.mark.parametrize("rows", [6, 700])
def test_the_smallest_uniform_draws_the_first_kept_token(vocab, size, rows):
    # light tokens lie before the heavy ones, by up to 2^-100 of the largest weight
    z = torch.arange(size, device="cuda", dtype=F32) * (69.0 / size) - 69.0
    x = z.expand(rows, size).clone()
    x[1] = x[1].flip(0)
    x[2] = x[2].roll(size // 2)
    x[3, 0] = -float("inf")
    x[4] = (x[4] / 8).round() * 8
    u = torch.zeros(rows, device="cuda")
    for f in (dict(), dict(top_k=size // 2), dict(top_k=150), dict(top_k=250), dict(top_k=800),
              dict(top_k=1000, top_p=0.999999), dict(top_k=2000), dict(min_p=1e-25),
              dict(top_k=900, min_p=1e-20)):
        got = vocab.sample_tokens(x, u, **f)
        for r in (0, 1, 2, 3, 4, rows - 1):
            y = x[r].double()
            order = y.argsort(descending=True, stable=True)
            n = int((y > -float("inf")).sum())
            if f.get("top_k"):
                n = min(n, f["top_k"])
            w = (y - y.max()).exp()
            run = w[order[:n]].cumsum(0)
            if "top_p" in f:
                p = float(torch.tensor(f["top_p"], dtype=F32))
                n = min(n, 1 + int((run < p * run[-1]).sum()))
            if "min_p" in f:
                m = float(torch.tensor(f["min_p"], dtype=F32))
                n = min(n, int((w >= m).sum()))
            # the definition: the first token whose running mass exceeds 0
            assert int(got.tokens[r]) == int(order[:n].min()), (r, f)
            assert int(got.kept[r]) == n, (r, f)
