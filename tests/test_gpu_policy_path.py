"""The policy's and the update's operators where the framework calls them: games played straight from a network's policy, the training
step with the loss from logits and with clipped gradients, and all of them in one loop."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

from test_gpu_policy_sample import _want  # noqa: E402
from test_gpu_selfplay import HashServe  # noqa: E402


def test_games_from_the_policy_alone():
    from muzero_amd import arena
    from muzero_amd.env import BatchedEnv
    n, t = 24, 0.5
    u = torch.from_numpy(np.random.default_rng(4).random((60, n))).cuda()
    nets = (HashServe("hash"), HashServe("sat"))
    got = arena.play_games(*nets, n, num_simulations=0, temperature=t, u=u)
    env = BatchedEnv(n)
    hw, hb = torch.zeros((61, n), dtype=torch.int64, device="cuda"), torch.zeros((61, n), dtype=torch.int64, device="cuda")
    hw[0], hb[0] = env.white, env.black
    for k in range(60):
        probs = nets[k % 2].initial(arena.controller_image(hw, hb, k, n))[1]
        want = _want(probs.log(), u[k], legal=env.legal, temperature=t)
        live = ~env.done.bool()
        acts = got.actions[k]
        assert all(a == w for a, w, l in zip(acts.tolist(), want, live.tolist()) if l), k
        env.step(acts.clone())
        hw[k + 1], hb[k + 1] = env.white, env.black
    assert got.white_score.tolist() == [bin(w & (2 ** 64 - 1)).count("1") for w in env.white.tolist()]


def _batch(B, K, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.rand(s, device="cuda", generator=g)   # noqa: E731
    pi = r(K + 1, B, 65) ** 8
    return ((r(B, 9, 8, 8) < 0.3).float(), (r(K, B, 2, 8, 8) < 0.1).float(), 2 * r(K + 1, B) - 1, pi / pi.sum(2, keepdim=True))


def _net(seed=3):
    from muzero_amd.network import Network
    torch.manual_seed(seed)
    return Network().cuda().train()


def _grads(net, batch, **kw):
    """the gradients that update_weights steps with, and its losses (a learning rate of 0 leaves the weights)"""
    from muzero_amd import train as T
    T.LOG = None
    opt = torch.optim.SGD(net.parameters(), lr=0.0)
    bucket = T.FlatGradBucket(net.parameters())
    losses = T.update_weights(opt, net, batch, bucket, **kw)
    return bucket.flat.clone(), [float(x) for x in losses]


@pytest.mark.parametrize("hip", [False, "x3"])
def test_training_step_with_the_loss_from_logits(hip):
    """log(softmax(x)) in two operations and in one: the losses and the gradients at the logits agree to about 100 roundings (6e-6); the rest of the
    backward pass is the same, and 1e-3 of the gradient's norm leaves it a hundredfold"""
    net, batch = _net(), _batch(32, 3, 1)
    a, la = _grads(net, batch, hip_convs=hip)
    b, lb = _grads(net, batch, hip_convs=hip, policy_from_logits=True)
    assert all(abs(p - q) <= 1e-5 * max(1.0, abs(p)) for p, q in zip(la, lb))
    assert (a - b).norm().item() <= 1e-3 * a.norm().item()


def test_training_step_with_clipped_gradients():
    net, batch = _net(), _batch(16, 2, 2)
    a, _ = _grads(net, batch)
    norm = a.double().norm().item()
    b, _ = _grads(net, batch, max_grad_norm=0.25 * norm)
    assert abs(b.double().norm().item() - 0.25 * norm) <= 1e-3 * norm        # the backward pass itself may sum in another order
    assert (b - 0.25 * a).norm().item() <= 1e-3 * norm
    c, _ = _grads(net, batch, max_grad_norm=4.0 * norm)
    assert (c - a).norm().item() <= 1e-3 * norm
    from muzero_amd import train as T
    net.zero_grad(set_to_none=True)                                            # without a bucket: the parameters' own gradients
    T.update_weights(torch.optim.SGD(net.parameters(), lr=0.0), net, batch, max_grad_norm=0.25 * norm)
    d = torch.cat([p.grad.reshape(-1) for p in net.parameters()])
    assert (d - b).norm().item() <= 1e-3 * norm


def test_a_probability_that_underflows():
    """200 below the others: f32 softmax gives 0, its logarithm -inf, and 0 targets times that NaN; from logits it is an ordinary row"""
    net, batch = _net(), _batch(8, 1, 3)
    pi = batch[3].clone()
    pi[..., 5] = 0.0
    batch = (*batch[:3], pi)
    with torch.no_grad():
        net.prediction.policy_head[-2].bias[5] = -200.0
    b, lb = _grads(net, batch, policy_from_logits=True)
    a, la = _grads(net, batch)                             # second: its step (0 times a NaN) spoils the weights
    assert not np.isfinite(la[0]) and np.isfinite(lb).all() and bool(b.isfinite().all())


def test_options_that_do_not_go_together():
    from muzero_amd import train as T
    net = _net()
    with pytest.raises(ValueError, match="amp_dtype"):
        T.update_weights(torch.optim.SGD(net.parameters(), lr=0.0), net, _batch(2, 1, 1), amp_dtype=torch.bfloat16, policy_from_logits=True)


def test_play_learn_and_clip_together():
    """policy play feeds nothing here: the loop's own self-play does; then the trained network plays from its policy"""
    from muzero_amd import arena, config
    from muzero_amd import train as T
    from muzero_amd.loop import MuZeroLoop
    T.LOG = None
    loop = MuZeroLoop(16, num_simulations=4, window_size=32, batch_size=16, max_grad_norm=0.5, policy_from_logits=True, train_convs="hip")
    before = [p.detach().clone() for p in loop.network.parameters()]
    losses = loop.generation(train_steps=3)
    assert len(losses) == 3 and all(bool(x.isfinite()) for pair in losses for x in pair)
    assert loop.bucket.flat.double().norm().item() <= 0.5 * (1 + 1e-5)
    assert any(not torch.equal(a, b) for a, b in zip(before, loop.network.parameters()))
    r = arena.play_games(loop.infer, loop.infer, 16, num_simulations=0)
    assert r.actions.shape == (config.max_moves, 16) and int(r.actions.max()) <= 64
    total = r.white_score + r.black_score
    assert bool((total >= 4).all()) and bool((total <= 64).all())
