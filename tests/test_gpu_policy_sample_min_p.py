"""min-p of more than 1 in one row counts as 1: where every mass rounds to 1 in 64 bits nothing is dropped, in rows of any length."""
import pytest
import torch

from test_gpu_policy_sample import _want

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kw", [dict(), dict(top_k=300), dict(top_p=0.75), dict(top_k=300, top_p=0.75)], ids=str)
@pytest.mark.parametrize("v", [65, 500, 1500, 3000, 7000, 9001, 50000])
def test_masses_that_round_to_one(v, kw):
    """at a temperature of 1e30 the masses of logits some units apart are 1 - 1e-30: 1"""
    from muzero_amd.policy import sample_actions
    g = torch.Generator(device="cuda").manual_seed(v)
    x = torch.randn(6, v, device="cuda", generator=g) * 3
    min_p = torch.tensor([2.0, 1.0, 0.5, 1e30, 0.0, float("nan")], device="cuda")
    u = torch.tensor([0.1, 0.3, 0.51, 0.77, 0.9, 0.99], dtype=torch.float64, device="cuda")
    got = sample_actions(x, u, temperature=1e30, min_p=min_p, **kw).tolist()
    assert got == _want(x, u, temperature=1e30, min_p=torch.tensor([1.0, 1.0, 0.5, 1.0, 0.0, 0.0]), **kw)
    if "top_p" not in kw:                      # one value for all rows
        assert sample_actions(x, u, temperature=1e30, min_p=1.0, **kw).tolist() == _want(x, u, temperature=1e30, min_p=1.0, **kw)


@pytest.mark.parametrize("v", [65, 500, 1500, 3000, 7000, 50000])
def test_at_ordinary_temperatures_only_the_best_stay(v):
    from muzero_amd.policy import sample_actions
    x = torch.randn(3, v, device="cuda", generator=torch.Generator(device="cuda").manual_seed(v))
    x[:, 3::v // 5] = 9.0                      # five or six equals ahead of the others
    u = torch.tensor([0.0, 0.5, 0.999], dtype=torch.float64, device="cuda")
    min_p = torch.tensor([2.0, 1.0, 7.5], device="cuda")
    assert sample_actions(x, u, min_p=min_p).tolist() == _want(x, u, min_p=1.0)
