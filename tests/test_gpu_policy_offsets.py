"""Offsets that pass 32 bits: the rows and tensors that lie behind the first 2^31 elements."""
import pytest
import torch

from test_gpu_policy_sample import _want

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kw", [dict(top_k=40, top_p=0.9), dict(top_p=0.95, temperature=0.8), dict(temperature=2.0), dict(top_p=0.9, temperature=3.0)], ids=str)
def test_sampling_from_the_last_rows(kw):
    from muzero_amd.policy import sample_actions
    n, v = 16500, 131072                                    # 2.16e9 elements
    x = torch.empty(n, v, dtype=torch.bfloat16, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(3)
    piece = (2.5 * torch.randn(500, v, device="cuda", generator=g)).to(torch.bfloat16)
    for a in range(0, n, 500):
        x[a:a + 500] = piece.roll(a // 7, 1)
    legal = torch.ones(n, v, dtype=torch.bool, device="cuda")
    legal[:, ::3] = False
    u = torch.rand(n, dtype=torch.float64, device="cuda", generator=g)
    at = [0, 1, 8191, 16382, 16383, 16384, 16385, 16498, 16499]
    assert sample_actions(x, u, **kw)[at].tolist() == _want(x[at], u[at], **kw)
    assert sample_actions(x, u, legal=legal, **kw)[at].tolist() == _want(x[at], u[at], legal=legal[at], **kw)


def test_short_rows_far_apart():
    """65 actions cut out of rows that are 2^26 apart"""
    from muzero_amd.policy import cross_entropy, sample_actions
    wide = torch.zeros(40, 1 << 26, dtype=torch.bfloat16, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(4)
    some = torch.randn(40, 65, device="cuda", generator=g).to(torch.bfloat16)
    wide[:, 7:72] = some
    x, u = wide[:, 7:72], torch.rand(40, dtype=torch.float64, device="cuda", generator=g)
    assert torch.equal(sample_actions(x, u, top_p=0.9), sample_actions(some, u, top_p=0.9))
    t = torch.rand(40, 65, device="cuda", generator=g)
    a, b = x.detach().requires_grad_(), some.detach().requires_grad_()
    la, lb = cross_entropy(a, t), cross_entropy(b, t)
    assert torch.equal(la, lb) and torch.equal(torch.autograd.grad(la, a)[0], torch.autograd.grad(lb, b)[0])


def test_a_gradient_of_more_than_2_31_elements():
    """every element is a power of two: the norm is exact, and so are the scaled values"""
    from muzero_amd.gradnorm import clip_grad_norm, grad_norm
    n = (1 << 31) + 4099
    t = torch.full((n,), 0.5, dtype=torch.bfloat16, device="cuda")
    t[-4099:] = 2.0
    want = ((1 << 31) * 0.25 + 4099 * 4.0) ** 0.5
    assert abs(grad_norm(t).double().item() - want) <= 2.0 ** -24 * want
    out = torch.zeros(n, dtype=torch.float32, device="cuda")
    clip_grad_norm(t, 1.0, out=out)
    scale = out[0] * 2.0
    assert abs(scale.double().item() - 1.0 / (want + 1e-6)) <= 2.0 ** -23 / want
    assert bool((out[:-4099] == scale * 0.5).all()) and bool((out[-4099:] == scale * 2.0).all())
