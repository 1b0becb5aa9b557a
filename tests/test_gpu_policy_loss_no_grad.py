"""The cross-entropy where no gradient is asked for: none is allocated or written, also where the logits are a leaf that requires one."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("n, v", [(20000, 65), (4000, 500), (600, 5003), (40, 70001), (3, 400001)])
def test_under_no_grad(n, v, reduction):
    from muzero_amd.policy import cross_entropy
    g = torch.Generator(device="cuda").manual_seed(v)
    x = torch.randn(n, v, device="cuda", generator=g).requires_grad_()
    t = torch.rand(n, v, device="cuda", generator=g)
    want = cross_entropy(x, t, reduction=reduction)
    assert want.requires_grad
    want = want.detach()
    for mode in (torch.no_grad, torch.inference_mode):
        with mode():
            torch.cuda.synchronize()
            torch.cuda.reset_peak_memory_stats()
            held = torch.cuda.memory_allocated()
            got = cross_entropy(x, t, reduction=reduction)
            assert torch.cuda.max_memory_allocated() - held < x.numel()     # a quarter of a gradient
        assert not got.requires_grad and torch.equal(got, want)
    assert torch.equal(cross_entropy(x.detach(), t, reduction=reduction), want)
    with torch.no_grad():
        with torch.enable_grad():
            loss = cross_entropy(x, t, reduction=reduction)
    assert torch.autograd.grad(loss.sum(), x)[0].shape == x.shape
