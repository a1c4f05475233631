"""What DesignEngine.resample takes as uniforms; the scored rows are stand-ins, so
that no GPU is needed to refuse."""
import numpy as np
import pytest
import torch

from hikoboshi_b200 import DesignEngine, HkbError


class Scored(DesignEngine):
    """An engine whose rows are given: two proteins of [3, 4] and [2, 5] positions."""

    def __init__(self, device):
        self.rows = torch.randn(22, 21, generator=torch.Generator().manual_seed(1)).to(device)

    def _scored_rows(self, coords, sources, tokens, orders, seeds):
        return self.rows, [(3, 4), (2, 5)]


def draw(uniforms, device="cpu"):
    return Scored(device).resample([], [], [], uniforms, temperature=0.7, top_p=0.9)


@pytest.mark.parametrize("uniforms,text", [
    ([np.zeros((3, 4))], "per position"), ([np.zeros((3, 4)), np.zeros((2, 4))], "per position"),
    ([np.zeros((4, 3)), np.zeros((2, 5))], "per position"),           # transposed
    ([np.zeros((3, 4)), np.zeros((5, 2))], "per position"),
    ([np.zeros((3, 4)), np.zeros((1, 10))], "per position"),
    ([np.full((3, 4), -1e-9), np.zeros((2, 5))], "0 to 1"),
    ([np.zeros((3, 4)), np.full((2, 5), 1.5)], "0 to 1"),
    ([np.zeros((3, 4)), np.full((2, 5), np.nan)], "0 to 1"),
])
def test_unfit_uniforms_are_refused(uniforms, text):
    with pytest.raises(HkbError) as e:
        draw(uniforms)
    assert e.value.code == 1 and text in e.value.detail


@pytest.mark.gpu
def test_flat_uniforms_are_the_same_draw():
    rng = np.random.default_rng(1)
    us = [rng.random((3, 4)), rng.random((2, 5))]
    us[0][0, 0], us[1][0, 0] = 0.0, 1.0
    for a, b in zip(draw(us, "cuda"), draw([u.reshape(-1) for u in us], "cuda")):
        assert all((x == y).all() and x.shape == y.shape for x, y in zip(a, b))
        assert (a[0] >= 0).all()
