"""Sampling an action from logits against the definition in 64 bits on the host: the answers have to be equal.  Where the definition leaves
a rounding open (a draw within 1e-12 of the border of two actions) no test draws: the uniforms are given, and ties are made of values
whose masses are exact."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def _row(x, ok, u, temperature, top_k, top_p, min_p):
    free = np.flatnonzero(ok & ~(x == -np.inf))
    if not free.size or np.isnan(x[free]).any() or (x[free] == np.inf).any() or math.isnan(temperature) or temperature == math.inf:
        return -1
    free = free[np.argsort(-x[free], kind="stable")]
    if temperature <= 0:
        return free[0]
    m = x[free[0]]
    if top_k > 0:
        free = free[:top_k]
    w = np.exp((x[free] - m) / temperature)
    keep = len(free)
    if top_p < 1:
        before = np.concatenate(([0.0], np.cumsum(w)[:-1]))
        keep = int((before < max(top_p, 0.0) * w.sum()).sum())
    keep = max(1, min(keep, int((w >= min(min_p, 1.0)).sum())))
    kept = np.sort(free[:keep])
    cum = np.cumsum(np.exp((x[kept] - m) / temperature))
    return kept[min(int(np.searchsorted(cum, u * cum[-1], side="right")), keep - 1)]


def _boards(legal):
    b = legal.cpu().numpy().astype(np.uint64)
    ok = ((b[:, None] >> np.arange(64, dtype=np.uint64)) & np.uint64(1)).astype(bool)
    return np.concatenate([ok, (b == 0)[:, None]], 1)


def _want(x, u, legal=None, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    n, v = x.shape
    xs, us = x.detach().double().cpu().numpy(), u.cpu().numpy()
    ok = np.ones((n, v), bool) if legal is None else legal.cpu().numpy() if legal.dim() == 2 else _boards(legal)
    per = [p.cpu().tolist() if torch.is_tensor(p) else [p] * n for p in (temperature, top_k, top_p, min_p)]
    return [int(_row(xs[i], ok[i], us[i], *(p[i] for p in per))) for i in range(n)]


def _uniforms(n, seed):
    u = torch.rand(n, dtype=torch.float64, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed))
    u[0] = 0.0
    if n > 1:
        u[1] = 1.0 - 1e-9
    return u


def _check(x, u, **kw):
    from muzero_amd.policy import sample_actions
    got = sample_actions(x, u, **kw)
    assert got.dtype == torch.int32 and got.shape == (x.shape[0],)
    want = _want(x, u, **kw)
    assert got.tolist() == want, [(i, a, b) for i, (a, b) in enumerate(zip(got.tolist(), want)) if a != b][:10]
    return got


SETTINGS = [dict(), dict(temperature=0.0), dict(temperature=0.25), dict(top_k=1), dict(top_k=5), dict(top_p=0.9), dict(top_p=0.3, temperature=1.7), dict(min_p=0.05),
            dict(top_k=40, top_p=0.8, temperature=0.7), dict(top_k=300, top_p=0.95, min_p=0.01), dict(top_p=0.97, min_p=0.2), dict(top_p=0.0), dict(min_p=1.0),
            dict(top_k=10 ** 9, top_p=0.999), dict(top_k=2500, top_p=0.5, temperature=2.0), dict(top_k=15000, top_p=0.99, temperature=3.0), dict(min_p=1e-4, temperature=2.0), dict(top_p=0.999999, temperature=3.0)]
SHAPES = [(1, 1), (5, 2), (3, 63), (9, 64), (64, 65), (5, 128), (5, 129), (7, 500), (4, 512), (5, 513), (3, 1000), (6, 2047), (3, 2048), (3, 2049), (4, 4096), (3, 4097), (5, 5003), (2, 8192), (3, 8193), (3, 32768), (2, 100003), (2, 131072)]


@pytest.mark.parametrize("kw", SETTINGS, ids=str)
@pytest.mark.parametrize("n, v", SHAPES)
@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=str)
def test_answers_are_the_definitions(n, v, dtype, kw):
    g = torch.Generator(device="cuda").manual_seed(n * 31 + v)
    x = (2.5 * torch.randn(n, v, device="cuda", generator=g)).to(dtype)
    u = _uniforms(n, v)
    _check(x, u, **kw)
    legal = torch.rand(n, v, device="cuda", generator=g) < 0.6
    legal[n // 2] = False                                  # a row that its mask leaves empty
    pad = torch.full((n, v + 3), math.nan, dtype=dtype, device="cuda")
    pad[:, 1:1 + v] = x.masked_fill(~legal, math.nan)        # rows of a wider buffer; what is not legal holds a NaN
    mask = torch.ones(n, v + 5, dtype=torch.bool, device="cuda")
    mask[:, 3:3 + v] = legal
    got = _check(pad[:, 1:1 + v], u, legal=mask[:, 3:3 + v], **kw)
    assert got[n // 2].item() == -1


@pytest.mark.parametrize("kw", SETTINGS[:9], ids=str)
def test_boards_of_legal_moves(kw):
    g = torch.Generator(device="cuda").manual_seed(8)
    x = torch.randn(300, 65, device="cuda", generator=g)
    legal = torch.randint(-2 ** 62, 2 ** 62, (300,), device="cuda", generator=g) & torch.randint(-2 ** 62, 2 ** 62, (300,), device="cuda", generator=g)
    legal[7] = 0
    legal[8] = -2 ** 63
    got = _check(x, _uniforms(300, 1), legal=legal, **kw)
    assert got[7].item() == 64 and got[8].item() == 63


@pytest.mark.parametrize("v", [65, 500, 1024, 4096, 6000, 40000])
def test_equal_logits_go_to_the_lower_index(v):
    g = torch.Generator(device="cuda").manual_seed(v)
    x = torch.zeros(8, v, device="cuda")
    x[4:] = torch.randint(0, 3, (4, v), device="cuda", generator=g).float() * math.log(2.0)   # masses 1, 1/2, 1/4 to a rounding
    x[7, ::2] = -0.0                                       # equal to +0
    u = _uniforms(8, v)
    for kw in (dict(temperature=0.0), dict(top_k=1), dict(top_k=7), dict(top_k=v - 1), dict(min_p=1.0), dict(min_p=0.4)):
        _check(x, u, **kw)
    e = torch.zeros(6, 2 ** int(math.log2(v)), device="cuda")    # equal masses: the share p ends exactly on a border
    for p in (0.5, 0.25, 0.75, 2.0 ** -6):
        got = _check(e, _uniforms(6, 3), top_p=p)
        assert max(got.tolist()) < p * e.shape[1]
    for p in (0.3, 0.61, 0.9):
        _check(x, u, top_p=p)
        _check(x, u, top_p=p, top_k=v // 2)


@pytest.mark.parametrize("v", [65, 500, 1500, 3000, 7000, 50000])
def test_settings_of_their_own_for_every_row(v):
    g = torch.Generator(device="cuda").manual_seed(v + 1)
    n = 24
    x = 3 * torch.randn(n, v, device="cuda", generator=g)
    r = lambda: torch.rand(n, device="cuda", generator=g)   # noqa: E731
    t, k, p, mp = 2 * r(), torch.randint(-3, 60, (n,), device="cuda", generator=g, dtype=torch.int32), r(), 0.3 * r()
    t[0], t[1], t[2], t[3] = 0.0, -1.0, math.nan, math.inf
    p[4], p[5], mp[6], mp[7], k[8], t[9] = 1.5, -0.5, -1.0, 2.0, 10 ** 9, 1e-40
    _check(x, _uniforms(n, 2), temperature=t, top_k=k, top_p=p, min_p=mp)
    _check(x, _uniforms(n, 2), temperature=t)
    _check(x, _uniforms(n, 2), top_k=k, top_p=0.9)
    _check(x, _uniforms(n, 2), top_p=p)


@pytest.mark.parametrize("v", [65, 500, 1500, 3000, 7000, 50000])
def test_infinities_nan_and_extreme_logits(v):
    x = torch.zeros(9, v, device="cuda")
    x[0, 3] = math.nan
    x[1, 3] = -math.nan
    x[2, v - 1] = math.inf
    x[3] = -math.inf                                     # nothing that could be played
    x[4] = -math.inf
    x[4, v - 2] = -1e30                                  # one action alone
    x[5] = torch.finfo(F32).min
    x[6] = torch.finfo(F32).min
    x[6, 5] = torch.finfo(F32).max
    x[7] = torch.linspace(-1e-38, 1e-38, v, device="cuda")
    x[8] = torch.linspace(-3e4, 3e4, v, device="cuda")
    u = _uniforms(9, 4)
    for kw in (dict(), dict(temperature=0.0), dict(top_k=3), dict(top_p=0.5), dict(min_p=0.5), dict(top_k=9, top_p=0.5, min_p=0.1)):
        got = _check(x, u, **kw).tolist()
        assert got[:5] == [-1, -1, -1, -1, v - 2] and got[6] == 5
    for t in (1e-30, 1e-3, 1e30):
        _check(x[:7], u[:7], temperature=t)


@pytest.mark.parametrize("v", [65, 600, 9000])
def test_uniforms_outside_their_range(v):
    from muzero_amd.policy import sample_actions
    x = torch.zeros(4, v, device="cuda")
    u = torch.tensor([-1.0, 1.0, 7.0, math.nan], dtype=torch.float64, device="cuda")
    assert sample_actions(x, u).tolist() == [0, v - 1, v - 1, v - 1]


def test_frequencies_follow_the_distribution():
    """a regular grid of uniforms visits every kept action in proportion to its mass, to one draw at each border"""
    from muzero_amd.policy import sample_actions
    v, n = 600, 20000
    x = torch.randn(1, v, device="cuda", generator=torch.Generator(device="cuda").manual_seed(5)) * 2
    u = (torch.arange(n, dtype=torch.float64, device="cuda") + 0.5) / n
    got = sample_actions(x.expand(n, v), u, temperature=0.8)
    p = (x[0].double() / 0.8).softmax(0)
    assert ((torch.bincount(got.long(), minlength=v) - n * p).abs() <= 1.0 + 1e-6).all()
    assert bool((got[1:] >= got[:-1]).all())


@pytest.mark.parametrize("kw", SETTINGS, ids=str)
@pytest.mark.parametrize("v, dtype", [(9000, F32), (20011, BF16), (6001, F16)], ids=str)
def test_more_rows_than_the_card_has_cus(v, dtype, kw):
    n = 300 if v > 8192 else 600
    x = (2.5 * torch.randn(n, v, device="cuda", generator=torch.Generator(device="cuda").manual_seed(v))).to(dtype)
    from muzero_amd.policy import sample_actions
    u = _uniforms(n, 12)
    got = sample_actions(x, u, **kw)
    at = list(range(0, n, 23))
    assert got[at].tolist() == _want(x[at], u[at], **kw)


@pytest.mark.parametrize("k", [200, 700, 1000, 2048, 2049, 4096, 4097])
@pytest.mark.parametrize("kind", ["spread", "integers", "one peak", "few legal", "equal", "huge", "steps"])
@pytest.mark.parametrize("n, v, dtype", [(3, 8193, F32), (3, 65537, F32), (2, 131072, BF16), (300, 9001, F16)], ids=str)
def test_many_of_the_best_in_long_rows(n, v, dtype, kind, k):
    """the k-th largest far inside the row, among equal ones, behind one far ahead of the others, or not there"""
    from muzero_amd.policy import sample_actions
    g = torch.Generator(device="cuda").manual_seed(v + k)
    x, legal = torch.randn(n, v, device="cuda", generator=g) * 2, None
    if kind == "integers":
        x = x.round()
    elif kind == "one peak":
        x[:, 77] = 40.0
    elif kind == "few legal":
        legal = torch.zeros(n, v, dtype=torch.bool, device="cuda")
        legal[:, 5::v // 600] = True
    elif kind == "equal":
        x.zero_()
    elif kind == "huge":
        x[:, 5] = 6e4
        x[:, 9] = -6e4
    elif kind == "steps":                        # sorted: the best are next to each other
        x = x.sort(dim=1).values
    x, u = x.to(dtype), _uniforms(n, k)
    at = list(range(0, n, max(1, n // 9)))
    for kw in (dict(), dict(top_p=0.8, temperature=2.0), dict(min_p=0.03)):
        got = sample_actions(x, u, top_k=k, legal=legal, **kw)
        assert got[at].tolist() == _want(x[at], u[at], legal=None if legal is None else legal[at], top_k=k, **kw), kw


@pytest.mark.parametrize("kw", [dict(), dict(top_k=60), dict(top_k=1000), dict(top_p=0.9), dict(min_p=1e-9)], ids=str)
@pytest.mark.parametrize("v", [65, 400, 2000, 5000, 9001, 131072])
def test_a_uniform_of_zero_takes_no_action_whose_mass_is_zero(v, kw):
    """e^-2000 is 0 in 64 bits; e^-600 is not"""
    x, u = torch.zeros(2, v, device="cuda"), torch.zeros(2, dtype=torch.float64, device="cuda")
    x[0, v - 2], x[1, v - 2] = 2000.0, 600.0
    got = _check(x, u, **kw).tolist()
    assert got == [v - 2, 0 if "top_p" not in kw and "min_p" not in kw else v - 2]


def test_many_rows_and_the_largest_vocabulary():
    g = torch.Generator(device="cuda").manual_seed(9)
    x = torch.randn(1, 2 ** 19, device="cuda", generator=g) * 3
    for kw in (dict(), dict(top_p=0.9), dict(top_k=100, top_p=0.9), dict(top_k=20000)):
        _check(x, _uniforms(1, 1) + 0.37, **kw)
    y = torch.randn(70000, 8200, device="cuda", generator=g, dtype=F32).to(F16)      # more rows than one pair of launches takes
    u = _uniforms(70000, 6)
    from muzero_amd.policy import sample_actions
    k = torch.randint(1, 50, (70000,), device="cuda", generator=g, dtype=torch.int32)
    got = sample_actions(y, u, top_k=k)
    at = list(range(0, 70000, 997)) + list(range(65520, 65550)) + [69999]
    assert got[at].tolist() == _want(y[at], u[at], top_k=k[at])


def test_same_answers_on_other_streams_and_in_graphs():
    from muzero_amd.policy import sample_actions
    g = torch.Generator(device="cuda").manual_seed(10)
    sets = [(torch.randn(n, v, device="cuda", generator=g) * 3, _uniforms(n, n)) for n, v in ((256, 65), (30, 9000), (4, 131072))]
    kw = dict(temperature=0.9, top_p=0.9)
    want = [sample_actions(x, u, **kw) for x, u in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = []
    for _ in range(3):
        for st, (x, u) in zip(streams, sets):
            with torch.cuda.stream(st):
                got.append(sample_actions(x, u, **kw))
    torch.cuda.synchronize()
    assert all(torch.equal(a, want[i % 3]) for i, a in enumerate(got))
    graphs = []
    for x, u in sets:
        out = torch.empty(x.shape[0], dtype=torch.int32, device="cuda")
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            assert sample_actions(x, u, out=out, **kw) is out
        graphs.append((gr, x, u, out))
    for k in range(3):
        for _, x, u, _ in graphs:
            x.mul_(0.9)
            u.mul_(0.95)
        for gr, *_ in graphs:
            gr.replay()
        torch.cuda.synchronize()
        for _, x, u, out in graphs:
            assert torch.equal(out, sample_actions(x, u, **kw))


def test_refusals():
    from muzero_amd import _lib as L
    from muzero_amd.policy import sample_actions
    x, u = torch.zeros(4, 65, device="cuda"), torch.zeros(4, dtype=torch.float64, device="cuda")
    for a, b, kw in ((x.double(), u, {}), (x[0], u, {}), (x.t(), u, {}), (x[:, ::2], u, {}), (x, u.float(), {}), (x, u[:3], {}), (x, u.cpu(), {}), (x[:, :0], u, {}),
                     (x, u, dict(legal=torch.ones(4, 64, dtype=torch.bool, device="cuda"))), (x, u, dict(legal=torch.ones(4, 65, device="cuda"))),
                     (x[:, :64], u, dict(legal=torch.ones(4, dtype=torch.int64, device="cuda"))), (x, u, dict(temperature=-1.0)), (x, u, dict(temperature=math.nan)),
                     (x, u, dict(top_k=-1)), (x, u, dict(top_k=2.5)), (x, u, dict(top_p=1.01)), (x, u, dict(min_p=-0.1)), (x, u, dict(min_p=math.nan)),
                     (x, u, dict(temperature=torch.ones(4, dtype=torch.float64, device="cuda"))), (x, u, dict(top_k=torch.ones(4, dtype=torch.int64, device="cuda"))),
                     (x, u, dict(top_p=torch.ones(3, device="cuda"))), (x, u, dict(out=torch.empty(4, dtype=torch.int64, device="cuda"))),
                     (x, u, dict(out=torch.empty(3, dtype=torch.int32, device="cuda")))):
        with pytest.raises(L.MzError):
            sample_actions(a, b, **kw)
    assert sample_actions(x[:0], u[:0]).shape == (0,)
