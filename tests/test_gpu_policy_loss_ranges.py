"""The cross-entropy's rows in chunks where its launches are cut: more rows than one pair of launches takes, and chunks of more than 8192 actions.

Tolerances as in test_gpu_policy_loss.py, with STEPS for these sizes: a lane's share of a chunk is at most 65536 / 256 = 256 actions, in runs of 4 or 8 (at most 64
of them, each 8 additions and a join of 5 roundings), and 8 + 9 + 8 joins of lanes, waves and chunks follow: 64 x 13 + 25 x 5 < 1000."""
import math

import pytest
import torch

import test_gpu_policy_loss as base

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def test_more_rows_than_one_pair_of_launches_takes():
    """rows that begin one element after each other in one buffer: all different, without 6 GB of them"""
    from muzero_amd.policy import cross_entropy
    n, v = 65540, 32771                       # 16-bit logits beside f32 targets: the longest rows held in registers have 32768
    g = torch.Generator(device="cuda").manual_seed(4)
    x = (torch.randn(n + v, device="cuda", generator=g) * 3).to(F16).as_strided((n, v), (1, 1)).requires_grad_()
    t = torch.rand(n + v, device="cuda", generator=g).div_(v).as_strided((n, v), (1, 1))
    w = torch.rand(n, device="cuda", generator=g) + 0.5
    w[::7] = 0.0
    rows = cross_entropy(x, t, weight=w, reduction="none")
    go = torch.linspace(-2, 3, n, device="cuda")
    got, = torch.autograd.grad(rows, x, go)
    loss = cross_entropy(x.detach(), t, weight=w)
    total, tol = 0.0, 0.0
    for a in range(0, n, 1024):
        b = min(n, a + 1024)
        ref, grad, rtol, gtol, _ = base._reference(x[a:b], t[a:b], w[a:b], None)
        assert bool(((rows[a:b].double() - ref).abs() <= rtol + 2 * base.U * ref.abs() + 1e-40).all()), a
        s = go[a:b].double()[:, None]
        base._check_grad(got[a:b], grad * s, gtol * s.abs(), 1.0, F16)
        total, tol = total + ref.sum().item(), tol + rtol.sum().item()
    assert abs(loss.double().item() - total / n) <= tol / n + base.U * abs(total / n)


@pytest.mark.parametrize("pair", [(F32, F32), (BF16, BF16), (F16, F32)], ids=str)
@pytest.mark.parametrize("n, v", [(2, 2 ** 21 + 2049), (17, 2 ** 21 + 5), (1, 2 ** 24 - 3), (2, 2 ** 24)])
@pytest.mark.parametrize("legal, pad, weight", [("none", 0, False), ("bool", 5, True)])
def test_chunks_of_many_actions(n, v, pair, legal, pad, weight, monkeypatch):
    from muzero_amd.policy import cross_entropy
    monkeypatch.setattr(base, "STEPS", 1000)
    x, t, w, lm = base._inputs(n, v, *pair, legal, pad, weight, seed=n + v)
    rows, grad, rtol, gtol, _ = base._reference(x, t, w, lm)
    loss = cross_entropy(x, t, weight=w, legal=lm)
    assert math.isfinite(loss.item()) and abs(loss.double().item() - rows.mean().item()) <= rtol.mean().item() + base.U * abs(rows.mean().item()) + 1e-40
    base._check_grad(torch.autograd.grad(loss, x)[0], grad, gtol, 1.0 / n, pair[0])


@pytest.mark.parametrize("n", [4_000_003, (1 << 22) - 1])
def test_as_many_rows_as_are_taken(n):
    from muzero_amd.policy import cross_entropy
    x, t, w, lm = base._inputs(n, 5, BF16, F32, "none", 0, True, seed=1)
    rows, grad, rtol, gtol, _ = base._reference(x, t, w, lm)
    loss = cross_entropy(x, t, weight=w)
    assert abs(loss.double().item() - rows.mean().item()) <= rtol.mean().item() + base.U * abs(rows.mean().item())
    base._check_grad(torch.autograd.grad(loss, x)[0], grad, gtol, 1.0 / n, BF16)
