"""A second derivative of the cross-entropy is refused however it is asked for: over the whole graph, or only towards chosen inputs, of the logits or of
what scales the loss.  Leaving it out would give the first-order part alone, without a word."""
import contextlib

import pytest
import torch

pytestmark = pytest.mark.gpu


def _graph(hooks=False, reduction="mean", scale=True):
    from muzero_amd.policy import cross_entropy
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(6, 65, device="cuda", generator=g).requires_grad_()
    w = torch.randn(65, 65, device="cuda", generator=g).requires_grad_()
    t = torch.rand(6, 65, device="cuda", generator=g)
    s = torch.tensor(1.5, device="cuda", requires_grad=True)
    with torch.autograd.graph.save_on_cpu() if hooks else contextlib.nullcontext():
        rows = cross_entropy(x @ w, t, reduction=reduction)
        loss = (rows * s if scale else rows).sum()
    return x, w, s, loss


@pytest.mark.parametrize("hooks", [False, True])
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_towards_chosen_inputs(reduction, hooks):
    x, w, s, loss = _graph(hooks, reduction)
    first, = torch.autograd.grad(loss, x, retain_graph=True)
    g, = torch.autograd.grad(loss, x, create_graph=True)
    assert torch.equal(g, first)
    for wrt in (x, w, s):
        with pytest.raises(RuntimeError, match="no second derivative"):
            torch.autograd.grad(loss + g.square().sum(), wrt, retain_graph=True)
    with pytest.raises(RuntimeError, match="no second derivative"):
        (loss + g.square().sum()).backward(inputs=[w], retain_graph=True)
    with pytest.raises(RuntimeError, match="no second derivative"):
        g.sum().backward(retain_graph=True)
    again, = torch.autograd.grad(loss, x, retain_graph=True)        # the first one is there as before
    assert torch.equal(again, first)


def test_an_unscaled_loss():
    """the gradient that the forward pass left is handed out; it depends on the logits all the same"""
    x, w, _, loss = _graph(scale=False)
    g, = torch.autograd.grad(loss, w, create_graph=True)
    with pytest.raises(RuntimeError, match="no second derivative"):
        torch.autograd.grad(g.square().sum(), x, retain_graph=True)
    with pytest.raises(RuntimeError, match="no second derivative"):
        torch.autograd.grad(loss + g.square().sum(), w)


def test_inputs_that_are_computed_again():
    """checkpointing hands out each saved tensor once"""
    from torch.utils.checkpoint import checkpoint
    from muzero_amd.policy import cross_entropy
    g = torch.Generator(device="cuda").manual_seed(4)
    x = torch.randn(6, 65, device="cuda", generator=g).requires_grad_()
    t = torch.rand(6, 65, device="cuda", generator=g)
    want, = torch.autograd.grad(cross_entropy(x * 2.0, t), x)
    loss = checkpoint(lambda y: cross_entropy(y * 2.0, t), x, use_reentrant=False)
    got, = torch.autograd.grad(loss, x, create_graph=True)
    assert torch.equal(got, want)
    with pytest.raises(RuntimeError, match="no second derivative"):
        torch.autograd.grad(got.square().sum(), x)
