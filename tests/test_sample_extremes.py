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
