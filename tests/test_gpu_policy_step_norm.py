"""The norm that a clipped training step had, kept where the step's other number, network.steps, is."""
import pytest
import torch

from test_gpu_policy_path import _batch, _grads, _net

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bucketed", [True, False])
def test_the_norm_of_the_last_step(bucketed):
    from muzero_amd import train as T
    net, batch = _net(), _batch(16, 2, 2)
    flat, _ = _grads(net, batch)
    want = flat.double().norm().item()
    assert not hasattr(net, "grad_norm")                       # an unclipped step has none
    net.zero_grad(set_to_none=True)
    bucket = T.FlatGradBucket(net.parameters()) if bucketed else None
    T.update_weights(torch.optim.SGD(net.parameters(), lr=0.0), net, batch, bucket, max_grad_norm=0.1 * want)
    norm = net.grad_norm
    assert norm.dim() == 0 and norm.is_cuda and not norm.requires_grad
    assert abs(norm.item() - want) <= 1e-3 * want              # the backward pass itself may sum in another order
    after = torch.cat([p.grad.reshape(-1) for p in net.parameters()]).double().norm().item()
    assert abs(after - 0.1 * want) <= 1e-3 * want


def test_a_step_of_infinite_gradients_can_be_seen():
    from muzero_amd import train as T
    net, (image, actions, values, policies) = _net(), _batch(4, 1, 3)
    values = values.clone()
    values[0, 0] = float("inf")
    T.update_weights(torch.optim.SGD(net.parameters(), lr=0.0), net, (image, actions, values, policies), T.FlatGradBucket(net.parameters()), max_grad_norm=1.0)
    assert not bool(net.grad_norm.isfinite())
