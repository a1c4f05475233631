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


def test_results_other_than_the_loss_are_detached():
    x, u = X.clone().requires_grad_(), torch.zeros(0)
    top = vocab.top_logits(x, 4)
    drawn = vocab.sample_tokens(x, u)
    both = vocab.distill_loss_and_grad(x, V, T)
    assert not any(a.requires_grad for a in (*top, *drawn, *both))
    # a teacher's tensors are constants
    v = V.clone().requires_grad_()
    norm = torch.zeros(0, requires_grad=True)
    assert not vocab.distill_loss(X, v, T, teacher_log_norm=norm).requires_grad
    loss = vocab.distill_loss(x, v, T, teacher_log_norm=norm)
    gx, gv, gn = torch.autograd.grad(loss.sum(), (x, v, norm), allow_unused=True)
    assert gx is not None and gv is None and gn is None


@pytest.mark.parametrize("transform", [
    lambda f: torch.func.vmap(f)(torch.zeros(2, 3, 21), torch.zeros(2, 3, 4),
                                 torch.zeros(2, 3, 4, dtype=torch.int32)),
    lambda f: torch.func.grad(lambda x: f(x, V, T).sum())(X),
    lambda f: torch.func.jvp(lambda x: f(x, V, T), (X,), (X,)),
    lambda f: torch.compile(lambda x: f(x, V, T), fullgraph=True, backend="eager")(X),
], ids=["vmap", "grad", "jvp", "compile"])
def test_transforms_raise(transform):
    with pytest.raises(RuntimeError):
        transform(vocab.distill_loss)


@pytest.mark.gpu
def test_a_backward_pass_alone_is_refused_in_a_capture():
    x = torch.randn(4, 50, device="cuda")
    v, t = x.topk(3)
    t, w = t.int(), torch.ones(4, device="cuda")
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        z = x.clone().requires_grad_()
        loss = vocab.distill_loss(z, v, t)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        with pytest.raises(RuntimeError, match="cannot be captured"):
            torch.autograd.grad(loss, z, w, retain_graph=True)
        _, inside = vocab.distill_loss_and_grad(x, v, t, row_weights=w)
    graph.replay()
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):  # the eager graph is as it was
        (after,) = torch.autograd.grad(loss, z, w)
    torch.cuda.synchronize()
    assert torch.equal(inside, after)
