"""Games straight from a policy that puts (nearly) all of its mass on a move that is not legal: the f32 probabilities of the legal ones underflow, their logits
do not."""
import numpy as np
import pytest
import torch

from test_gpu_policy_sample import _want

pytestmark = pytest.mark.gpu
CORNER = 0                                       # not legal in the opening


def _network(gap, seed=3):
    from muzero_amd.network import Network
    torch.manual_seed(seed)
    net = Network()
    with torch.no_grad():
        net.prediction.policy_head[-2].weight.mul_(8.0)
        net.prediction.policy_head[-2].bias[CORNER] += gap
    return net


def _logits(engine, hidden):
    head = engine.net.prediction.policy_head[:-1].float()      # the serving weights are exact in f32; called last: it changes the engine
    return head(hidden.float())


@pytest.mark.parametrize("kind", ["f32", "bf16", "f32 hip_x3", "f16 miopen"])
def test_moves_come_from_the_logits(kind):
    from muzero_amd import arena, config
    from muzero_amd.env import BatchedEnv
    from muzero_amd.network import InferenceEngine
    n, t = 32, 1.0
    kw = {"f32": dict(dtype=torch.float32), "bf16": dict(dtype=torch.bfloat16), "f32 hip_x3": dict(dtype=torch.float32, channels_last=False, tower="hip_x3"),
          "f16 miopen": dict(dtype=torch.float16)}[kind]
    engine = InferenceEngine(_network(300.0), n, **kw)
    u = torch.from_numpy(np.random.default_rng(5).random((config.max_moves, n))).cuda()
    got = arena.play_games(engine, engine, n, num_simulations=0, temperature=t, u=u)
    assert int(got.actions.max()) <= 64
    env = BatchedEnv(n)
    hw, hb = env.white.clone().view(1, n), env.black.clone().view(1, n)
    image = arena.controller_image(hw, hb, 0, n, engine.dtype)
    _, probs, hidden = engine.initial(image)
    assert not bool(probs[:, [19, 26, 37, 44, 20, 29, 34, 43]].any())              # whichever four of these are legal: nothing of them is left
    want = _want(_logits(engine, hidden).detach(), u[0], legal=env.legal, temperature=t)
    assert got.actions[0].tolist() == want and len(set(want)) > 1


def test_a_network_that_gives_probabilities_alone():
    """legal moves of no mass are equally likely; a NaN is still refused as a move"""
    from muzero_amd import _lib as L
    from muzero_amd import arena, config

    class Serve:
        dtype = torch.float32

        def __init__(self, fill):
            self.fill = fill

        def initial(self, image):
            n = image.shape[0]
            p = torch.full((n, 65), self.fill, device="cuda")
            p[:, CORNER] = 1.0
            return torch.zeros(n, device="cuda"), p, torch.zeros((n, 8, 8, 8), device="cuda")

    from muzero_amd.env import BatchedEnv
    n = 48
    u = torch.from_numpy(np.random.default_rng(6).random((config.max_moves, n))).cuda()
    got = arena.play_games(Serve(0.0), Serve(0.0), n, num_simulations=0, u=u)
    env = BatchedEnv(n)
    assert got.actions[0].tolist() == _want(torch.zeros(n, 65, device="cuda"), u[0], legal=env.legal, temperature=0.25)
    with pytest.raises(L.MzError, match="illegal"):
        arena.play_games(Serve(float("nan")), Serve(0.0), n, num_simulations=0, u=u)


def test_finished_games_record_the_pass():
    """whatever the policy of a game is once that is over (its 60th move was no pass): here a NaN from then on"""
    from muzero_amd import arena, config

    class Serve:
        dtype = torch.float32
        moves = 0

        def initial(self, image):
            n = image.shape[0]
            Serve.moves += 1
            p = torch.full((n, 65), 1.0 / 65, device="cuda")
            if Serve.moves > config.max_moves:
                p[over] = float("nan")
            return torch.zeros(n, device="cuda"), p, torch.zeros((n, 8, 8, 8), device="cuda")

    n, t = 64, config.max_moves + 1
    u = torch.from_numpy(np.random.default_rng(7).random((t, n))).cuda()
    first = arena.play_games(Serve(), Serve(), n, num_simulations=0, temperature=1.0, u=u)
    over = first.done.bool().cuda()
    assert bool(over.any())
    Serve.moves = 0
    got = arena.play_games(Serve(), Serve(), n, num_simulations=0, temperature=1.0, u=u, max_steps=t)
    assert torch.equal(got.actions[:-1], first.actions) and bool((got.actions[-1][over] == 64).all())


@pytest.mark.parametrize("kind", ["adapter", "f32", "bf16", "f32 hip_x3"])
def test_logits_are_those_of_the_served_policy(kind):
    """log softmax of the logits against the logarithm of the policy that came with the hidden states.  Two f32 chains of 8 + 128 + 128 products: each is wrong by
    at most 2^-24 of the terms' absolute sum per step, so 2 x 264 x 2^-24 of that together, and the two softmaxes and logarithms 32 x 2^-24 of 1 + |log p| more."""
    import copy
    from muzero_amd.network import InferenceEngine, policy_logits
    from muzero_amd.selfplay import NetworkAdapter
    net, n = _network(0.0), 64
    image = (torch.rand(n, 9, 8, 8, device="cuda", generator=torch.Generator(device="cuda").manual_seed(8)) < 0.3).float()
    engine = {"adapter": lambda: NetworkAdapter(net.cuda()), "f32": lambda: InferenceEngine(net, n, torch.float32), "bf16": lambda: InferenceEngine(net, n, torch.bfloat16),
              "f32 hip_x3": lambda: InferenceEngine(net, n, torch.float32, channels_last=False, tower="hip_x3")}[kind]()
    _, probs, hidden = engine.initial(image.to(engine.dtype))
    got = engine.policy_logits(hidden)
    assert got.dtype == torch.float32 and got.shape == (n, 65) and not got.requires_grad
    positive = copy.deepcopy(engine.net)
    for p in positive.parameters():
        p.requires_grad_(False).abs_()
    size = policy_logits(positive)(hidden.abs()).double().amax(1, keepdim=True)       # no term is larger
    want = probs.double().log()
    assert bool(((got.double().log_softmax(1) - want).abs() <= 2.0 ** -24 * (2 * 2 * 264 * size + 32 * (1 + want.abs()))).all())


def test_adapters_of_other_networks_and_copies_of_adapters():
    import copy
    import pickle
    from muzero_amd.selfplay import NetworkAdapter

    class Other:
        def initial_inference(self, image):
            n = image.shape[0]
            return torch.zeros(n, 1, device="cuda"), torch.full((n, 65), 1.0 / 65, device="cuda"), torch.zeros((n, 8, 8, 8), device="cuda")

    class Changed(torch.nn.Module):
        def forward(self, hidden):
            n = hidden.shape[0]
            return torch.full((n, 65), 1.0 / 65, device="cuda"), torch.zeros(n, 1, device="cuda")

    from muzero_amd import arena
    from muzero_amd.network import InferenceEngine
    assert not hasattr(NetworkAdapter(Other()), "policy_logits")
    arena.play_games(NetworkAdapter(Other()), NetworkAdapter(Other()), 4, num_simulations=0)
    engine = InferenceEngine(_network(0.0), 4, torch.float32)
    assert hasattr(engine, "policy_logits")
    engine.net.prediction = Changed()                       # a head of another form, served by the same engine
    assert not hasattr(engine, "policy_logits")
    arena.play_games(engine, engine, 4, num_simulations=0)
    adapter = NetworkAdapter(_network(0.0).cuda())
    hidden = torch.rand(3, 8, 8, 8, device="cuda")
    want = adapter.policy_logits(hidden)
    for twin in (copy.deepcopy(adapter), pickle.loads(pickle.dumps(adapter))):
        assert torch.equal(twin.policy_logits(hidden), want)
        with torch.no_grad():
            twin.net.prediction.policy_head[-2].bias.add_(1.0)          # its own network, not the first one's
        assert not torch.equal(twin.policy_logits(hidden), want) and torch.equal(adapter.policy_logits(hidden), want)
