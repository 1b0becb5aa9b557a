"""The policy's cross-entropy and its gradient against the formulas in 64 bits.

Tolerances, with u = 2^-24 and d = x - m: exp(d) carries |d| u from the rounding of d and 2 u of its own, a sum of positive terms one u per
addition of its longest chain.  A lane adds at most 64 terms, and at most 36 steps join lanes, waves and chunks, so STEPS = 100 covers every
path.  Row loss: u w (STEPS (T (|log z| + 1) + sum t |d|) + T max |d|), with the largest |d| among terms that weigh in z (those below 2^-24 of it
add nothing).  Gradient: u s (T p (STEPS + |d|) + 4 |g| / s), half a step of its type, half the smallest subnormal."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
U, STEPS = 2.0 ** -24, 100
HALF = {F32: 0.0, BF16: 2.0 ** -8, F16: 2.0 ** -11}
TINY = {F32: 2.0 ** -149, BF16: 2.0 ** -133, F16: 2.0 ** -24}


def _allowed(legal, n, v):
    if legal is None:
        return torch.ones((n, v), dtype=torch.bool, device="cuda")
    if legal.dim() == 2:
        return legal
    return torch.stack([(legal >> i & 1).bool() for i in range(64)] + [legal == 0], 1)


def _reference(x, t, w, legal):
    """64-bit rows, gradient for a loss gradient of 1 and no mean, and their tolerances in units of w"""
    n, v = x.shape
    ok = _allowed(legal, n, v)
    x = torch.where(ok, x.detach().double(), -math.inf)
    t = torch.where(ok, t.double(), 0.0)
    w = torch.ones(n, dtype=torch.float64, device="cuda") if w is None else w.double()
    m = x.max(1, keepdim=True).values
    live = (m > -math.inf) & (w != 0)[:, None]
    d = torch.where(live, x - m, 0.0)
    e = torch.where(live, d.exp(), 0.0)
    z = torch.where(live, e.sum(1, keepdim=True), 1.0)
    T = t.sum(1, keepdim=True)
    td = torch.where(t != 0, t * d, 0.0).sum(1, keepdim=True)
    rows = torch.where(live, w[:, None] * (T * z.log() - td), 0.0)[:, 0]
    p = e / z
    grad = torch.where(live & ok, w[:, None] * (T * p - t), 0.0)
    dz = torch.where(p > U, d.abs(), 0.0).amax(1, keepdim=True)
    rtol = U * w[:, None] * (STEPS * (T * (z.log().abs() + 1) + td.abs()) + T * dz)
    gtol = U * w[:, None] * T * p * (STEPS + torch.where(p > 0, d.abs(), 0.0))
    return rows, grad, rtol[:, 0], gtol, live[:, 0]


def _check_grad(got, grad, gtol, scale, dtype):
    assert got.dtype == dtype and got.shape == grad.shape
    ref = grad * scale
    tol = gtol * scale + ref.abs() * (4 * U + HALF[dtype]) + TINY[dtype]
    bad = (got.double() - ref).abs() > tol
    assert not bool(bad.any()), ((got.double() - ref).abs() / tol).max().item()


def _inputs(n, v, dtype, tdtype, legal, pad, weight, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = (3.0 * torch.randn(n, v + pad, device="cuda", generator=g)).to(dtype)[:, pad // 2:pad // 2 + v]
    t = torch.randn(n, v + pad, device="cuda", generator=g).mul(2).softmax(1).to(tdtype)[:, pad - pad // 2:pad - pad // 2 + v]
    lm = None
    if legal == "bool":
        lm = torch.rand(n, v + pad, device="cuda", generator=g)[:, pad // 2:pad // 2 + v] < 0.7
        lm[n // 2] = False
        if pad:
            lm = torch.nn.functional.pad(lm, (1, pad - 1))[:, 1:1 + v]
    elif legal == "board":
        lm = torch.randint(-2 ** 62, 2 ** 62, (n,), device="cuda", generator=g) & torch.randint(-2 ** 62, 2 ** 62, (n,), device="cuda", generator=g)
        lm[n // 3] = 0
        lm[0] |= -2 ** 63
    w = None
    if weight:
        w = torch.rand(n, device="cuda", generator=g) + 0.5
        w[::3] = 0.0
    return x.detach().requires_grad_(), t, w, lm


SHAPES = [(1, 1), (1, 65), (6, 2), (3, 64), (7, 128), (4, 129), (9, 512), (6, 513), (5, 1000), (3, 2049), (4, 4097), (3, 8191), (2, 16384), (3, 16391), (2, 40000),
          (130, 20000), (129, 33001), (131, 65536), (129, 70001), (2, 131072), (1, 200001), (17, 140001), (3, 70000)]


@pytest.mark.parametrize("pair", [(F32, F32), (BF16, BF16), (BF16, F32), (F16, F16), (F16, F32)], ids=str)
@pytest.mark.parametrize("n, v", SHAPES)
@pytest.mark.parametrize("legal, pad, weight", [("none", 0, False), ("bool", 5, True)])
def test_loss_and_gradient_match_the_formula(n, v, pair, legal, pad, weight):
    from muzero_amd.policy import cross_entropy
    x, t, w, lm = _inputs(n, v, *pair, legal, pad, weight, seed=n * 7 + v)
    rows, grad, rtol, gtol, _ = _reference(x, t, w, lm)
    loss = cross_entropy(x, t, weight=w, legal=lm)
    assert loss.dtype == F32 and loss.dim() == 0
    assert abs(loss.double().item() - rows.mean().item()) <= rtol.mean().item() + U * abs(rows.mean().item()) + 1e-40
    _check_grad(torch.autograd.grad(loss, x)[0], grad, gtol, 1.0 / n, pair[0])
    per_row = cross_entropy(x, t, weight=w, legal=lm, reduction="none")
    assert per_row.shape == (n,) and bool(((per_row.double() - rows).abs() <= rtol + 2 * U * rows.abs() + 1e-40).all())
    go = torch.linspace(-2, 3, n, device="cuda")
    got, = torch.autograd.grad(per_row, x, go)
    _check_grad(got, grad * go.double()[:, None], gtol * go.abs().double()[:, None], 1.0, pair[0])
    with torch.no_grad():                                  # without a gradient: the same loss
        assert torch.equal(cross_entropy(x, t, weight=w, legal=lm), loss)


@pytest.mark.parametrize("pair", [(F32, F32), (F16, F32)], ids=str)
def test_boards_of_legal_moves(pair):
    from muzero_amd.policy import cross_entropy
    x, t, w, lm = _inputs(517, 65, *pair, "board", 0, True, seed=11)
    rows, grad, rtol, gtol, _ = _reference(x, t, w, lm)
    loss = cross_entropy(x, t, weight=w, legal=lm, reduction="sum")
    assert abs(loss.double().item() - rows.sum().item()) <= rtol.sum().item() + U * abs(rows.sum().item())
    _check_grad(torch.autograd.grad(loss, x)[0], grad, gtol, 1.0, pair[0])
    same = cross_entropy(x, t, weight=w, legal=_allowed(lm, 517, 65), reduction="sum")
    assert torch.equal(same, loss)


def test_many_long_rows():
    from muzero_amd.policy import cross_entropy
    x, t, w, lm = _inputs(230, 140001, F32, F32, "none", 0, True, seed=5) 
    rows, grad, rtol, gtol, _ = _reference(x, t, w, lm)
    loss = cross_entropy(x, t, weight=w)
    assert abs(loss.double().item() - rows.mean().item()) <= rtol.mean().item() + U * abs(rows.mean().item())
    _check_grad(torch.autograd.grad(loss, x)[0], grad, gtol, 1.0 / 230, F32)


@pytest.mark.parametrize("v", [65, 300, 5000, 40000])
def test_what_is_not_legal_is_never_used(v):
    from muzero_amd.policy import cross_entropy
    x, t, _, lm = _inputs(6, v, F32, F32, "bool", 0, False, seed=v)
    lm[0, 0] = True
    clean = cross_entropy(x, t, legal=lm, reduction="none")
    want, = torch.autograd.grad(clean.sum(), x)
    for bad in (math.nan, math.inf, -math.inf, torch.finfo(F32).max, torch.finfo(F32).min):
        xb = torch.where(lm, x.detach(), bad).requires_grad_()
        tb = torch.where(lm, t, bad)
        rows = cross_entropy(xb, tb, legal=lm, reduction="none")
        assert torch.equal(rows, clean)
        assert torch.equal(torch.autograd.grad(rows.sum(), xb)[0], want)
    assert clean[3].item() == 0.0 and not bool(want[3].any()) and not bool(want[~lm].any())
    w = torch.ones(6, device="cuda")
    w[2] = 0.0                                                # a padding row may hold anything
    xb, tb = x.detach().clone(), t.clone()
    xb[2], tb[2] = math.nan, math.inf
    xb.requires_grad_()
    rows = cross_entropy(xb, tb, weight=w, legal=lm, reduction="none")
    got, = torch.autograd.grad(rows.sum(), xb)
    assert rows[2].item() == 0.0 and not bool(got[2].any())
    assert torch.equal(rows[3:], clean[3:]) and torch.equal(got[3:], want[3:])


@pytest.mark.parametrize("v", [65, 300, 5000, 40000])
def test_infinities_and_nan_follow_the_formula(v):
    from muzero_amd.policy import cross_entropy
    x = torch.zeros(6, v, device="cuda")
    t = torch.zeros(6, v, device="cuda")
    t[:, 1] = 1.0
    x[0, 0] = -math.inf                       # no target there: log(v - 1)
    x[1, 1] = -math.inf                       # the target itself: infinite
    x[2] = -math.inf                          # nothing that could be played: 0
    x[3, v - 1] = math.nan
    x[4, v - 1] = math.inf
    x[5] = torch.finfo(F32).min               # the lowest value of the type in every place: log v
    x.requires_grad_()
    rows = cross_entropy(x, t, reduction="none")
    g, = torch.autograd.grad(rows.sum(), x)
    assert abs(rows[0].item() - math.log(v - 1)) <= 100 * U * math.log(v) and rows[1].item() == math.inf and rows[2].item() == 0.0
    assert bool(rows[3].isnan()) and bool(rows[4].isnan()) and abs(rows[5].item() - math.log(v)) <= 100 * U * math.log(v)
    assert g[0, 0].item() == 0.0 and not bool(g[2].any()) and bool(g[3].isnan().all()) and bool(g[[0, 1, 2, 5]].isfinite().all())
    x = torch.full((1, v), math.nan, device="cuda")
    assert bool(cross_entropy(x, t[:1]).isnan())


def test_gradient_against_differences():
    """central differences of the loss itself: their truncation is at most h^2 / 6 times the third derivative (|p''| <= T / 8), their
    rounding the loss's tolerance over h"""
    from muzero_amd.policy import cross_entropy
    h = 2.0 ** -4
    for v in (5, 600):
        x, t, w, lm = _inputs(3, v, F32, F32, "bool", 0, False, seed=v)
        lm[1, 0] = True
        rows, _, rtol, _, _ = _reference(x, t, w, lm)
        g, = torch.autograd.grad(cross_entropy(x, t, legal=lm, reduction="sum"), x)
        for i in range(3):
            for j in range(0, v, max(1, v // 7)):
                s = torch.zeros_like(x)
                s[i, j] = h
                with torch.no_grad():
                    up, down = (cross_entropy(x + k * s, t, legal=lm, reduction="none")[i].double().item() for k in (1, -1))
                T = t[i].sum().item()
                tol = h * h / 6 * T / 8 + 2 * (rtol[i].item() + 2 * U * abs(rows[i].item())) / h + 4 * U * T / h
                assert abs((up - down) / (2 * h) - g[i, j].item()) <= tol


def test_a_loss_inside_a_larger_one():
    """the gradient of the loss is not 1: a scaled 16-bit loss whose unscaled gradient would underflow, a second pass over a kept graph, and a
    network in front of the logits"""
    from muzero_amd.policy import cross_entropy
    x, t, w, lm = _inputs(2000, 65, F16, F32, "none", 0, False, seed=2)
    rows, grad, rtol, gtol, _ = _reference(x, t, w, lm)
    loss = cross_entropy(x, t)
    first, = torch.autograd.grad(loss, x, retain_graph=True)
    kept = first.clone()
    scaled, = torch.autograd.grad(loss * 4096.0, x, retain_graph=True)
    _check_grad(scaled, grad, gtol, 4096.0 / 2000, F16)
    again, = torch.autograd.grad(loss, x)
    _check_grad(first, grad, gtol, 1.0 / 2000, F16)
    assert torch.equal(first, kept) and torch.equal(again, kept) and again.data_ptr() != first.data_ptr()
    x2 = x.detach().clone().requires_grad_()
    got, = torch.autograd.grad(cross_entropy(x2, t) * 4096.0, x2)              # the first pass over the graph already scaled
    assert torch.equal(got, scaled)
    lin = torch.nn.Linear(20, 65).cuda()
    f = torch.randn(33, 20, device="cuda")
    tt = torch.rand(33, 65, device="cuda")
    (cross_entropy(lin(f), tt) + lin(f).square().mean()).backward()
    a = lin.weight.grad.clone()
    lin.zero_grad()
    ((-tt * torch.log_softmax(lin(f), 1)).sum(1).mean() + lin(f).square().mean()).backward()
    assert (a - lin.weight.grad).abs().max().item() <= 1e-4 * a.abs().max().item()   # two f32 forms, 65 and 33 terms each: 100 roundings and the Linear's own


def test_changed_logits_are_noticed():
    from muzero_amd.policy import cross_entropy
    x, t, _, _ = _inputs(4, 65, F32, F32, "none", 0, False, seed=1)
    y = x * 1.0
    loss = cross_entropy(y, t)
    y.add_(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


@pytest.mark.parametrize("legal", ["none", "bool"])
@pytest.mark.parametrize("n, v", [(40, 65), (9, 5003), (3, 70001)])
def test_saved_tensors_that_come_back_elsewhere(n, v, legal):
    """between forward and backward the inputs are kept on the host, or computed again: other addresses and other strides"""
    from torch.utils.checkpoint import checkpoint
    from muzero_amd.policy import cross_entropy
    x, t, w, lm = _inputs(n, v, BF16, F32, legal, 7, True, seed=v)
    want, = torch.autograd.grad(cross_entropy(x, t, w, lm) * 3.0, x)
    leaf = x.detach().clone().requires_grad_()

    def loss(leaf):
        wide = torch.nn.functional.pad(leaf, (2, 5))
        return cross_entropy(wide[:, 2:2 + v], t.clone(), w.clone(), None if lm is None else lm.clone()) * 3.0

    with torch.autograd.graph.save_on_cpu():
        kept = loss(leaf)
    again = checkpoint(loss, leaf, use_reentrant=False)
    for total in (kept, again):
        junk = [torch.full((n, v + 7), math.nan, dtype=d, device="cuda") for d in (BF16, BF16, F32, F32)]   # where the inputs were
        got, = torch.autograd.grad(total, leaf)
        del junk
        assert torch.equal(got, want)


@pytest.mark.parametrize("v", [65, 5000, 70001])
def test_rows_that_share_their_memory(v):
    """one row of logits and one mask for all: their gradients add up"""
    from muzero_amd.policy import cross_entropy
    n = 5
    x, t, w, _ = _inputs(n, v, F32, F32, "none", 0, True, seed=v)
    one = x.detach()[:1].clone().requires_grad_()
    mask = (torch.rand(1, v, device="cuda") < 0.5).expand(n, v)
    rows, grad, rtol, gtol, _ = _reference(one.detach().expand(n, v), t, w, mask)
    loss = cross_entropy(one.expand(n, v), t, weight=w, legal=mask, reduction="sum")
    assert abs(loss.double().item() - rows.sum().item()) <= rtol.sum().item() + U * abs(rows.sum().item()) + 1e-40
    got, = torch.autograd.grad(loss, one)
    tol = gtol.sum(0) + (4 + n) * U * grad.abs().sum(0) + TINY[F32]
    assert bool(((got[0].double() - grad.sum(0)).abs() <= tol).all())


def test_a_second_derivative_is_refused():
    from muzero_amd.policy import cross_entropy
    x, t, _, _ = _inputs(4, 65, F32, F32, "none", 0, False, seed=3)
    want, = torch.autograd.grad(cross_entropy(x, t), x)
    got, = torch.autograd.grad(cross_entropy(x, t), x, create_graph=True)
    assert torch.equal(got, want)
    with pytest.raises(RuntimeError, match="no second derivative"):
        (got.square().sum() + x.sum()).backward()


def test_no_rows():
    from muzero_amd.policy import cross_entropy
    x = torch.zeros(0, 65, device="cuda", requires_grad=True)
    t = torch.zeros(0, 65, device="cuda")
    assert bool(cross_entropy(x, t).isnan()) and cross_entropy(x, t, reduction="none").shape == (0,)
    s = cross_entropy(x, t, reduction="sum")
    assert s.item() == 0.0 and torch.autograd.grad(s, x)[0].shape == (0, 65)


def test_streams_and_replayed_graphs():
    from muzero_amd.policy import cross_entropy
    sets = []
    for n, v in ((512, 65), (40, 5000), (3, 50000)):
        x, t, w, lm = _inputs(n, v, F32, F32, "none", 0, True, seed=v)
        sets.append((x, t, w))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    outs = []
    for _ in range(3):
        for st, (x, t, w) in zip(streams, sets):
            with torch.cuda.stream(st):
                loss = cross_entropy(x, t, weight=w)
                outs.append((loss.detach(), torch.autograd.grad(loss, x)[0], x, t, w))
    torch.cuda.synchronize()
    for loss, g, x, t, w in outs:
        rows, grad, rtol, gtol, _ = _reference(x, t, w, None)
        assert abs(loss.double().item() - rows.mean().item()) <= rtol.mean().item() + U * rows.mean().item()
        _check_grad(g, grad, gtol, 1.0 / x.shape[0], F32)
    outs = loss = g = None
    graphs = []
    for x, t, w in sets:
        x = x.detach().clone().requires_grad_()
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            loss = cross_entropy(x, t, weight=w)
            g, = torch.autograd.grad(loss, x)
        graphs.append((gr, x, t, w, loss.detach(), g))
    for k in range(3):
        for _, x, _, _, _, _ in graphs:
            x.data.mul_(0.8).add_(0.01)
        for gr, *_ in graphs:
            gr.replay()
        torch.cuda.synchronize()
        for _, x, t, w, loss, g in graphs:
            xx = x.detach().clone().requires_grad_()
            eager = cross_entropy(xx, t, weight=w)
            assert torch.equal(eager, loss) and torch.equal(torch.autograd.grad(eager, xx)[0], g)


def test_refusals():
    from muzero_amd import _lib as L
    from muzero_amd.policy import cross_entropy
    x, t = torch.zeros(4, 65, device="cuda"), torch.zeros(4, 65, device="cuda")
    for a, b, kw in ((x.double(), t.double(), {}), (x, t.half(), {}), (x.half(), t.bfloat16(), {}), (x[0], t[0], {}), (x, t[:3], {}), (x.t(), t.t(), {}), (x, t.cpu(), {}),
                     (x[:, ::2], t[:, :33], {}), (x[:, :0], t[:, :0], {}), (x, t, dict(weight=torch.ones(3, device="cuda"))), (x, t, dict(weight=torch.ones(4))),
                     (x, t, dict(weight=torch.ones(4, device="cuda").double())), (x, t, dict(legal=torch.ones(4, 64, dtype=torch.bool, device="cuda"))),
                     (x, t, dict(legal=torch.ones(4, 65, device="cuda"))), (x, t, dict(legal=torch.ones(3, dtype=torch.int64, device="cuda"))),
                     (x[:, :64], t[:, :64], dict(legal=torch.ones(4, dtype=torch.int64, device="cuda"))), (x, t, dict(legal=torch.ones(4, dtype=torch.int64))),
                     (x, t.clone().requires_grad_(), {}), (x, t, dict(reduction="max"))):
        with pytest.raises(L.MzError):
            cross_entropy(a, b, **kw)
