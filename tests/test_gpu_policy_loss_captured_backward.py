"""A backward pass of the cross-entropy that is captured without its forward pass: every replay computes the gradient for the factor that lies there then."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n, v", [(40, 65), (9, 5003), (3, 70001)])
def test_replays_with_other_factors(n, v):
    from muzero_amd.policy import cross_entropy
    g = torch.Generator(device="cuda").manual_seed(v)
    x = torch.randn(n, v, device="cuda", generator=g).requires_grad_()
    t = torch.rand(n, v, device="cuda", generator=g)
    go = torch.ones((), device="cuda")
    want = {}
    for f in (1.0, 4.0, -0.5):
        want[f], = torch.autograd.grad(cross_entropy(x, t), x, torch.full((), f, device="cuda"))
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        loss = cross_entropy(x, t)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            got, = torch.autograd.grad(loss, x, go, retain_graph=True)
    torch.cuda.synchronize()
    for f in (1.0, 4.0, 1.0, -0.5, 1.0):
        go.fill_(f)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want[f]), f
    again, = torch.autograd.grad(loss, x)                # the kept graph, eagerly: memory of its own
    torch.cuda.synchronize()
    assert torch.equal(again, want[1.0]) and again.data_ptr() != got.data_ptr()


@pytest.mark.parametrize("n, v", [(40, 65), (9, 5003), (3, 70001)])
def test_forward_and_backward_in_graphs_of_their_own(n, v):
    from muzero_amd.policy import cross_entropy
    g = torch.Generator(device="cuda").manual_seed(v)
    x = torch.randn(n, v, device="cuda", generator=g).requires_grad_()
    t = torch.rand(n, v, device="cuda", generator=g)
    go = torch.ones((), device="cuda")
    torch.cuda.synchronize()
    side, forward, backward = torch.cuda.Stream(), torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        with torch.cuda.graph(forward, stream=side):
            loss = cross_entropy(x, t)
        with torch.cuda.graph(backward, stream=side):
            got, = torch.autograd.grad(loss, x, go, retain_graph=True)
    torch.cuda.synchronize()
    for step in range(3):
        x.data.mul_(0.9)
        torch.cuda.synchronize()
        forward.replay()
        for f in (1.0, 4.0, 1.0):
            torch.cuda.synchronize()
            go.fill_(f)
            torch.cuda.synchronize()
            backward.replay()
            torch.cuda.synchronize()
            xx = x.detach().clone().requires_grad_()
            eager = cross_entropy(xx, t)
            assert torch.equal(loss, eager) and torch.equal(got, torch.autograd.grad(eager, xx, go.clone())[0]), (step, f)
