"""Host side of muzero_amd/policy.py without a GPU: what it refuses (no CPU fallback: host tensors raise), and the C entry points'
checks, which come before any launch."""
import ctypes as C

import pytest
import torch


def test_cross_entropy_refuses_host_tensors():
    from muzero_amd import _lib as L
    from muzero_amd import policy
    with pytest.raises(L.MzError, match="no CPU fallback"):
        policy.cross_entropy(torch.zeros(2, 65), torch.zeros(2, 65))


def _args(L, **kw):
    P = 1 << 40                                   # never read: every call below is refused on the host
    d = dict(logits=P, targets=P, loss=P, n=4, v=65, logits_stride=65, targets_stride=65, grad_stride=65, scale=0.25)
    d.update(kw)
    a = L.PolicyLossArgs()
    for k, v in d.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("kw, why", [
    (dict(n=-1), "n has to be"), (dict(n=1 << 22), "n has to be"), (dict(v=0), "v has to be"), (dict(v=(1 << 24) + 1), "v has to be"),
    (dict(dtype=3), "unknown dtype"), (dict(dtype=0, target_dtype=1), "targets have"), (dict(dtype=1, target_dtype=2), "targets have"),
    (dict(v=64, board=1 << 40), "needs v = 65"), (dict(board=1 << 40, allowed=1 << 40), "not both"), (dict(loss=None), "no output"),
    (dict(skip_one=1), "needs one grad_out"), (dict(skip_one=1, grad_out=1 << 40, grad_out_stride=1), "needs one grad_out"),
    (dict(skip_one=1, grad_out=1 << 40), "leaves the loss out"), (dict(grad_out_stride=2), "0 or 1"), (dict(logits=None), "null"),
    (dict(targets=None), "null"), (dict(logits=(1 << 40) + 2), "misaligned"), (dict(grad=(1 << 40) + 2), "misaligned"),
    (dict(logits_stride=-1), "negative"), (dict(grad=1 << 40, grad_stride=64), "overlap"),
])
def test_policy_loss_arguments_are_checked_before_any_launch(kw, why):
    from muzero_amd import _lib as L
    with pytest.raises(L.MzError, match=why):
        L.call("mz_policy_loss", C.byref(_args(L, **kw)), 1 << 40, 1 << 30, None)


def test_policy_loss_workspace_is_checked():
    from muzero_amd import _lib as L
    need = L.lib.mz_policy_loss_workspace_bytes(4, 65)
    assert need > 0
    for bad in ((-1, 65), (4, 0), (4, (1 << 24) + 1), (1 << 22, 65)):
        assert L.lib.mz_policy_loss_workspace_bytes(*bad) == -1
    for ws, nbytes, why in ((None, 1 << 30, "workspace"), ((1 << 40) + 8, 1 << 30, "misaligned"), (1 << 40, need - 1, "needed")):
        with pytest.raises(L.MzError, match=why):
            L.call("mz_policy_loss", C.byref(_args(L)), ws, nbytes, None)
    with pytest.raises(L.MzError, match="null arguments"):
        L.call("mz_policy_loss", None, 1 << 40, 1 << 30, None)
    L.call("mz_policy_loss", C.byref(_args(L, n=0, logits=None, targets=None)), None, 0, None)   # no rows: nothing to do


def test_sample_actions_refuses_host_tensors():
    from muzero_amd import _lib as L
    from muzero_amd import policy
    with pytest.raises(L.MzError, match="no CPU fallback"):
        policy.sample_actions(torch.zeros(2, 65), torch.zeros(2, dtype=torch.float64))


def _sample(L, **kw):
    P = 1 << 40                                   # never read: every call below is refused on the host
    d = dict(logits=P, u=P, action=P, n=4, v=10000, logits_stride=10000, temperature=1.0, top_p=1.0)
    d.update(kw)
    a = L.SampleArgs()
    for k, v in d.items():
        setattr(a, k, v)
    return a


NAN = float("nan")


@pytest.mark.parametrize("kw, why", [
    (dict(n=-1), "n has to be"), (dict(n=1 << 22), "n has to be"), (dict(v=0), "v has to be"), (dict(v=(1 << 19) + 1), "v has to be"), (dict(dtype=3), "unknown dtype"),
    (dict(v=64, board=1 << 40), "needs v = 65"), (dict(board=1 << 40, v=65, allowed=1 << 40), "not both"), (dict(temperature=-1.0), "temperature"),
    (dict(temperature=NAN), "temperature"), (dict(temperature=1e-31), "temperature"), (dict(temperature=float("inf")), "temperature"), (dict(top_k=-1), "top_k"),
    (dict(top_p=-0.1), "top_p"), (dict(top_p=1.1), "top_p"), (dict(top_p=NAN), "top_p"), (dict(min_p=-0.1), "min_p"), (dict(min_p=1.1), "min_p"), (dict(min_p=NAN), "min_p"),
    (dict(logits=None), "null"), (dict(u=None), "null"), (dict(action=None), "null"), (dict(logits=(1 << 40) + 2), "misaligned"), (dict(logits_stride=-1), "negative"),
    (dict(allowed=1 << 40, allowed_stride=-1), "negative"),
])
def test_sample_arguments_are_checked_before_any_launch(kw, why):
    from muzero_amd import _lib as L
    with pytest.raises(L.MzError, match=why):
        L.call("mz_sample_actions", C.byref(_sample(L, **kw)), 1 << 40, 1 << 30, None)


def test_sample_workspace_is_checked():
    from muzero_amd import _lib as L
    size = L.lib.mz_sample_actions_workspace_bytes
    assert size(4, 8192) == 0 and size(4, 8193) == 4 * 65 * 12 and size(513, 4096) == 0 and size(513, 4097) == 513 * 33 * 12
    for bad in ((-1, 65), (4, 0), (4, (1 << 19) + 1), (1 << 22, 65)):
        assert size(*bad) == -1
    for ws, nbytes, why in ((None, 1 << 30, "workspace"), ((1 << 40) + 4, 1 << 30, "misaligned"), (1 << 40, size(4, 10000) - 1, "needed")):
        with pytest.raises(L.MzError, match=why):
            L.call("mz_sample_actions", C.byref(_sample(L)), ws, nbytes, None)
    with pytest.raises(L.MzError, match="null arguments"):
        L.call("mz_sample_actions", None, 1 << 40, 1 << 30, None)
    L.call("mz_sample_actions", C.byref(_sample(L, n=0, logits=None, u=None, action=None)), None, 0, None)   # no rows: nothing to do


def test_training_options_need_the_gpu():
    from muzero_amd import train as T
    from muzero_amd.network import Network
    net = Network()
    opt = T.make_optimizer(net)
    for kw in (dict(max_grad_norm=1.0), dict(policy_from_logits=True)):
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            T.update_weights(opt, net, None, T.FlatGradBucket(net.parameters()), **kw)


def test_argument_structures_as_bytes():
    """policy.py packs the structures of include/muzero_amd.h itself: the same sizes and places as the ctypes ones"""
    from muzero_amd import _lib as L
    from muzero_amd import policy
    for pack, cls in ((policy._LOSS_ARGS, L.PolicyLossArgs), (policy._SAMPLE_ARGS, L.SampleArgs)):
        names = [f[0] for f in cls._fields_]
        values = [1.0 + k if t is C.c_double else k + 1 for k, (_, t) in enumerate(cls._fields_)]
        raw = pack(*values)
        assert len(raw) == C.sizeof(cls)
        a = cls.from_buffer_copy(raw)
        assert [getattr(a, k) for k in names] == values
