"""What autograd and torch's transforms get of the operators on vocabulary rows:
derivatives that they have, and no wrong ones."""
import pytest
import torch
import torch.autograd.forward_ad as forward_ad

from hikoboshi_b200 import HkbError, vocab

X, V = torch.zeros(0, 21), torch.zeros(0, 4)
T = torch.zeros(0, 4, dtype=torch.int32)


def test_forward_mode_is_refused_instead_of_dropping_the_tangent():
    with forward_ad.dual_level():
        for x in (X, X.clone().requires_grad_()):
            dual = forward_ad.make_dual(x, torch.ones_like(X))
            with pytest.raises(HkbError) as e:
                vocab.distill_loss(dual, V, T)
            assert e.value.code == 1 and "forward-mode" in e.value.detail
        # without a tangent the call is what it was
        assert vocab.distill_loss(X, V, T).shape == (0,)
