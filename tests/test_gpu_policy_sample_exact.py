"""Sampling where nothing is rounded: whole logits at the temperature 1 / ln 2, so that masses are powers of two, with shares, min-p and uniforms of few bits.  The cuts
fall exactly on borders, among many equals, and the answers have to be the definition's in every form of the operator."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16
T = 1.4426950408889634            # log2(e) / T is 1


def _row(x, u, k, p, min_p):
    order = np.argsort(-x, kind="stable")
    if k > 0:
        order = order[:k]
    w = np.exp2(x[order] - x[order[0]])
    keep = len(order)
    if p < 1:
        keep = int((np.cumsum(w) - w < p * w.sum()).sum())
    keep = max(1, min(keep, int((w >= min_p).sum())))
    kept = np.sort(order[:keep])
    cum = np.cumsum(np.exp2(x[kept] - x[order[0]]))
    return int(kept[min(int(np.searchsorted(cum, u * cum[-1], side="right")), keep - 1)])


@pytest.mark.parametrize("top", [1, 17])
@pytest.mark.parametrize("kind", ["p", "kp", "kpm", "m"])
@pytest.mark.parametrize("n, v", [(64, 65), (40, 300), (24, 512), (24, 700), (16, 2048), (12, 4096), (12, 8192), (9, 9001), (270, 8200), (6, 131072)])
@pytest.mark.parametrize("dtype", [F32, BF16], ids=str)
def test_cuts_exactly_on_borders(n, v, dtype, kind, top):
    from muzero_amd.policy import sample_actions
    rng = np.random.default_rng([n, v, top, len(kind)])
    x = rng.integers(0, top + 1, (n, v)) - rng.integers(0, 9, (n, 1))
    x[::4, rng.integers(0, v)] += 3                             # now and then one ahead of all
    x[1::4] = np.where(rng.random((len(x[1::4]), v)) < 0.98, x[1::4].min(axis=1, keepdims=True), x[1::4])      # and few above a flat floor
    k = rng.integers(1, max(2, min(v, 12000)), n) if "k" in kind else np.zeros(n, np.int64)
    k[::3] = np.minimum(k[::3], 40)
    p = rng.integers(1, 256, n) / 256.0 if "p" in kind else np.ones(n)
    min_p = 2.0 ** -rng.integers(0, top + 2, n) if "m" in kind else np.zeros(n)
    u = rng.integers(0, 1 << 20, n) / float(1 << 20)
    u[:2] = 0.0, 1.0 - 2.0 ** -20
    dev = lambda a, t: torch.tensor(a, device="cuda", dtype=t)   # noqa: E731
    got = sample_actions(dev(x, F32).to(dtype), dev(u, torch.float64), temperature=T, top_k=dev(k, torch.int32), top_p=dev(p, F32), min_p=dev(min_p, F32)).tolist()
    at = range(n) if n < 100 else range(0, n, 7)
    want = [_row(x[i].astype(np.float64), u[i], int(k[i]), float(p[i]), float(min_p[i])) for i in at]
    assert [got[i] for i in at] == want, [(i, got[i], b) for i, b in zip(at, want) if got[i] != b][:5]
