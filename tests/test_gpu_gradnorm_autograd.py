"""The gradient norm and clipping where their tensors carry a graph of their own: neither has a derivative, and a backward pass that needs one says so instead
of taking the norm and the factor for constants."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _pair():
    g = torch.Generator(device="cuda").manual_seed(2)
    a = torch.randn(300, device="cuda", generator=g).requires_grad_()
    b = torch.randn(7, 5, device="cuda", generator=g).requires_grad_()
    return a, b


def test_a_penalty_on_the_norm_is_refused():
    from muzero_amd.gradnorm import grad_norm
    a, b = _pair()
    grads = torch.autograd.grad((a ** 3).sum() + (b ** 2).sum() * a.sum(), (a, b), create_graph=True)
    norm = grad_norm(grads)
    want = torch.cat([g.detach().reshape(-1) for g in grads]).double().norm()
    assert abs(norm.detach().double().item() - want.item()) <= 2.0 ** -24 * (1 + 1e-6) * want.item()
    for wrt in (a, b):
        with pytest.raises(RuntimeError, match="no derivative"):
            torch.autograd.grad((a ** 2).sum() + (b ** 2).sum() + norm, wrt, retain_graph=True)
    with pytest.raises(RuntimeError, match="no derivative"):
        grad_norm([torch.ones(4, device="cuda"), a]).backward()
    with torch.no_grad():
        assert not grad_norm(grads).requires_grad
    assert not grad_norm([g.detach() for g in grads]).requires_grad


def test_what_was_scaled_in_place_has_no_derivative():
    from muzero_amd.gradnorm import clip_grad_norm
    a, b = _pair()
    y, z = a * 2.0, b + 1.0
    before = y.sum()                                     # used before: its gradient is what it was
    want = [t.detach() * (0.5 / (torch.cat([y.detach().reshape(-1), z.detach().reshape(-1)]).double().norm() + 1e-6)).clamp(max=1.0).float() for t in (y, z)]
    norm = clip_grad_norm([y, z], 0.5)
    assert all(bool(((g.detach() - w).abs() <= 3 * 2.0 ** -24 * w.abs() + 2.0 ** -149).all()) for g, w in zip((y, z), want))
    for loss, wrt in ((y.sum(), a), (z.sum() + b.sum(), b), (norm + a.sum(), a)):
        with pytest.raises(RuntimeError, match="no derivative"):
            torch.autograd.grad(loss, wrt, retain_graph=True)
    assert torch.equal(torch.autograd.grad(before, a)[0], torch.full_like(a, 2.0))
    y = a * 2.0
    clip_grad_norm([y[3:200]], 0.5)                      # a part of it
    with pytest.raises(RuntimeError, match="no derivative"):
        torch.autograd.grad(y[250] + a.sum(), a)
    y = a * 2.0
    with torch.no_grad():                                # as an optimiser does
        clip_grad_norm([y], 0.5)
    assert torch.equal(torch.autograd.grad(y.sum(), a)[0], torch.full_like(a, 2.0))


def test_outputs_beside_tensors_that_carry_a_graph():
    from muzero_amd import _lib as L
    from muzero_amd.gradnorm import clip_grad_norm
    a, _ = _pair()
    y, out = a * 2.0, torch.zeros(300, device="cuda")
    with pytest.raises(L.MzError, match="detach"):
        clip_grad_norm([y], 0.5, out=[out])
    assert not bool(out.any())
    with torch.no_grad():
        clip_grad_norm([y], 0.5, out=[out])
    assert abs(out.double().norm().item() - 0.5) <= 1e-5
    clip_grad_norm([y.detach()], 0.5, out=[out])
    assert not out.requires_grad


def test_leaves_and_gradients_as_before():
    """parameters are scaled as values, like in an optimiser's step; their gradients carry no graph"""
    from muzero_amd.gradnorm import clip_grad_norm, grad_norm
    a, b = _pair()
    (a.square().sum() + b.square().sum()).backward()
    norm = clip_grad_norm([a.grad, b.grad], 1e-2)
    assert not norm.requires_grad and abs(torch.cat([a.grad.reshape(-1), b.grad.reshape(-1)]).double().norm().item() - 1e-2) <= 1e-6
    assert not grad_norm([a.grad, b.grad]).requires_grad
    clip_grad_norm([a, b], 1e-2)
    assert a.is_leaf and b.is_leaf and abs(torch.cat([a.detach().reshape(-1), b.detach().reshape(-1)]).double().norm().item() - 1e-2) <= 1e-6


def test_views_that_autograd_takes_nothing_in_place_from():
    """torch refuses the pieces of a split, and this does before anything is scaled"""
    from muzero_amd.gradnorm import clip_grad_norm
    a, _ = _pair()
    y = a * 2.0
    kept = y.detach().clone()
    with pytest.raises(RuntimeError, match="view"):
        clip_grad_norm(list(torch.split(y, 100)), 0.5)
    assert torch.equal(y.detach(), kept)


def test_the_norm_that_clipping_returns_for_leaves():
    from muzero_amd.gradnorm import clip_grad_norm
    a, b = _pair()
    norm = clip_grad_norm([a, b], 1e-2)
    with pytest.raises(RuntimeError, match="no derivative"):
        torch.autograd.grad(a.sum() + norm, a)
    with torch.no_grad():
        assert not clip_grad_norm([a, b], 1e-2).requires_grad
