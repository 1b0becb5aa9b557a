"""Sampling where the share p ends far out: the best action holds nearly everything and the cut falls among many that hold 1e-13 of it each.

u = 1 answers the last kept action, so the answer is the kept set's size.  The peak's mass is 1, a tail action's w = e^-30 = 9.4e-14 = 843 x 2^-53, and p is put
half an action behind a border, so what may be wrong together is half of w, 421 x 2^-53.  p and its product with the total: 2 roundings of 2^-53.  The total: a
lane adds at most 16 values, and 40 steps join lanes, waves and groups, of which each is wrong by at most 2^-53: 56.  The polynomial of the groups' masses: 2e-12 of a
tail of 5e-8, 1e-19.  Equal tails are divided by one mass, so nothing else adds up: the answer is exact.  In tails that fall off by e^-0.5 (511 x 2^-53 at the end)
masses are added up as integers of 2^-61, half a unit wrong each: for 2^19 of them, all rounded one way, 2^-43 = 1024 x 2^-53.  (421 + 58 + 1024) / 511 < 3 actions."""
import math

import pytest
import torch

from test_gpu_policy_sample import _uniforms, _want

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
# rows, actions, legal ones beside the peak (0: all), top_k
CASES = [(2, 600, 0, 0), (3, 2048, 0, 0), (3, 4096, 0, 0), (2, 8192, 0, 0), (2, 8192, 0, 6000), (2, 131072, 5000, 0), (2, 131072, 5000, 3000), (2, 131072, 0, 0),
         (2, 131072, 0, 20000), (300, 9001, 0, 0), (300, 20000, 2500, 0), (1, 2 ** 19, 0, 0), (5, 512, 0, 0)]


def _legal(n, v, count, peak):
    if not count:
        return None
    ok = torch.zeros(n, v, dtype=torch.bool, device="cuda")
    ok[:, 1::v // count] = True
    ok[:, peak] = True
    return ok


def _kept(order, masses, share):
    """actions kept of `order` (best first), and p such that the cut falls half an action behind them"""
    total = math.fsum(masses)
    k = max(2, int(share * len(masses)))
    return order[:k], (math.fsum(masses[:k]) - 0.5 * masses[k - 1]) / total


@pytest.mark.parametrize("share", [0.3, 0.51, 0.9])
@pytest.mark.parametrize("n, v, count, top_k", CASES)
@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=str)
def test_a_cut_inside_a_tail_of_equals(n, v, count, top_k, dtype, share):
    from muzero_amd.policy import sample_actions
    peak = v // 3
    x = torch.full((n, v), -30.0, device="cuda")
    x[:, peak] = 0.0
    legal = _legal(n, v, count, peak)
    tail = [j for j in (range(v) if legal is None else legal[0].nonzero()[:, 0].tolist()) if j != peak]
    m = (top_k or len(tail) + 1) - 1                           # tail actions that top-k leaves
    kept, p = _kept([peak] + tail[:m], [1.0] + [math.exp(-30.0)] * m, share)
    got = sample_actions(x.to(dtype), torch.ones(n, dtype=torch.float64, device="cuda"), top_k=top_k, top_p=p, legal=legal)
    assert got.tolist() == [max(kept)] * n


@pytest.mark.parametrize("share", [0.3, 0.51, 0.9])
@pytest.mark.parametrize("n, v, count, top_k", CASES)
def test_a_cut_inside_a_tail_that_falls_off(n, v, count, top_k, share):
    """its logits fall by 1/2 in the order of the indices, the peak stands first"""
    from muzero_amd.policy import sample_actions
    x = -30.0 - 0.5 * torch.arange(v, device="cuda", dtype=F32).expand(n, v) / v
    x = x.clone()
    x[:, 0] = 0.0
    legal = _legal(n, v, count, 0)
    order = list(range(v)) if legal is None else legal[0].nonzero()[:, 0].tolist()
    if top_k:
        order = order[:top_k]
    xs = x[0].double().tolist()
    if len({xs[j] for j in order}) < len(order):               # equals, by f32's rounding, stay in the order of the indices: as written here
        assert all(xs[a] >= xs[b] for a, b in zip(order, order[1:]))
    kept, p = _kept(order, [math.exp(xs[j]) for j in order], share)
    got = sample_actions(x, torch.ones(n, dtype=torch.float64, device="cuda"), top_k=top_k, top_p=p, legal=legal)
    place = {j: i for i, j in enumerate(order)}
    assert all(j in place and abs(place[j] - (len(kept) - 1)) < 3 for j in got.tolist()), (got.tolist()[:4], kept[-1])


@pytest.mark.parametrize("v", [300, 3000, 8000, 70000])
def test_draws_of_a_uniform_in_its_range(v):
    """the same cut, u = 1 - 1e-9: the mass that u leaves beyond the answer is 1e-9 of the total, 10685 tail actions (at most all of them)"""
    from muzero_amd.policy import sample_actions
    x = torch.full((1, v), -30.0, device="cuda")
    x[:, 0] = 0.0
    kept, p = _kept(list(range(v)), [1.0] + [math.exp(-30.0)] * (v - 1), 0.9)
    got = sample_actions(x, torch.tensor([1.0 - 1e-9], dtype=torch.float64, device="cuda"), top_p=p).item()
    total = 1.0 + (len(kept) - 1) * math.exp(-30.0)
    want = max(0, math.floor(((1.0 - 1e-9) * total - 1.0) / math.exp(-30.0)) + 1)
    assert abs(got - want) <= 1          # u times the total and the cumulated masses: some 60 roundings of 2^-53, 843 of which are an action
