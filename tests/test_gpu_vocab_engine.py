"""The operators on vocabulary rows as the engine's own paths call them: scored
rows drawn anew, and a student that learns from an engine's answers.  With a
weight image of random values."""
import numpy as np
import pytest
import torch

from random_weights import random_weights
from vocab_reference import distill_row, sample_row, top_row

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", params=["fp32", "f16"])
def case(request):
    from hikoboshi_b200 import DesignEngine, synthetic_backbone
    backbones = [synthetic_backbone(3, 40), synthetic_backbone(4, 57)]
    coords, sources = [b[0] for b in backbones], [b[1] for b in backbones]
    rng = np.random.default_rng(1)
    tokens = [rng.integers(0, 21, (s, len(c))).astype(np.int32) for s, c in zip((3, 2), coords)]
    eng = DesignEngine(random_weights(5), precision=request.param)
    yield eng, coords, sources, tokens, eng.score(coords, sources, tokens, seeds=9)
    eng.close()


def test_resample_draws_from_the_scored_rows(case):
    eng, coords, sources, tokens, scored = case
    rng = np.random.default_rng(2)
    uniforms = [rng.random(t.shape) for t in tokens]
    got = eng.resample(coords, sources, tokens, uniforms, temperature=0.5, top_k=9, top_p=0.9,
                       min_p=0.02, seeds=9)
    assert len(got) == 2
    for (t, lp, kept), u, (rows, _, _) in zip(got, uniforms, scored):
        assert t.shape == lp.shape == kept.shape == u.shape
        for s in range(t.shape[0]):
            for i in range(t.shape[1]):
                token, want, n = sample_row(rows[s, i].astype(np.float64), u[s, i], 0.5, 9,
                                            float(np.float32(0.9)), float(np.float32(0.02)),
                                            drawn=int(t[s, i]))
                assert (t[s, i], kept[s, i]) == (token, n)
                assert abs(lp[s, i] - want) <= 2.0 ** -24 * abs(want) + 1e-12
    greedy = eng.resample(coords, sources, tokens, uniforms, temperature=0.0, seeds=9)
    for (t, lp, kept), (rows, _, _) in zip(greedy, scored):
        assert (t == rows.argmax(-1)).all() and (lp == 0).all() and (kept == 1).all()


def test_distill_targets_are_the_scored_rows_and_train_a_student(case):
    from hikoboshi_b200 import vocab
    eng, coords, sources, tokens, scored = case
    targets = eng.distill_targets(coords, sources, tokens, 6, temperature=2.0, seeds=9)
    for top, (rows, _, _) in zip(targets, scored):
        assert top.values.shape == (*rows.shape[:2], 6) and top.log_norm.shape == rows.shape[:2]
        for s in range(rows.shape[0]):
            for i in range(rows.shape[1]):
                order, norm, err = top_row(rows[s, i].astype(np.float64), 6, 2.0)
                assert (top.tokens[s, i].cpu().numpy() == order).all()
                assert (top.values[s, i].cpu().numpy() == rows[s, i][order]).all()
                assert abs(float(top.log_norm[s, i]) - norm) <= err
    # one step of a student on the targets: its gradient reaches its weights
    top = targets[0]
    gen = torch.Generator(device="cuda").manual_seed(3)
    hidden = torch.randn(*top.log_norm.shape, 16, generator=gen, device="cuda")
    weight = torch.randn(16, 21, generator=gen, device="cuda").requires_grad_()
    logits = hidden @ weight
    loss = vocab.distill_loss(logits, top.values, top.tokens, teacher_log_norm=top.log_norm,
                              temperature=2.0)
    loss.mean().backward()
    n = loss.numel()
    want, bound = torch.zeros(16, 21, dtype=torch.float64), torch.zeros(16, 21, dtype=torch.float64)
    for s in range(loss.shape[0]):
        for i in range(loss.shape[1]):
            x = logits[s, i].detach().double().cpu().numpy()
            value, g, lerr, gerr = distill_row(x, top.values[s, i].double().cpu().numpy(),
                                               top.tokens[s, i].cpu().numpy(),
                                               float(top.log_norm[s, i]), 2.0, torch.float32)
            assert abs(float(loss[s, i]) - value) <= lerr
            h = hidden[s, i].double().cpu()
            want += torch.outer(h, torch.from_numpy(g)) / n
            bound += torch.outer(h.abs(), torch.from_numpy(gerr + abs(g) * 2.0 ** -24)) / n
            # the product that carries it to the weights: TF32 is off, n terms
            bound += torch.outer(h.abs(), torch.from_numpy(abs(g))) * 2.0 ** -24 * n / n
    assert ((weight.grad.double().cpu() - want).abs() <= bound).all()


def test_resample_checks_its_uniforms(case):
    from hikoboshi_b200 import HkbError
    eng, coords, sources, tokens, _ = case
    with pytest.raises(HkbError) as e:
        eng.resample(coords, sources, tokens, [np.zeros((3, 40)), np.zeros((2, 56))])
    assert e.value.code == 1 and "uniforms" in e.value.detail
