"""The gradient norm and clipping against the formulas in 64 bits.

Tolerances: the norm is a 64-bit sum rounded once to f32 (half a step: 2^-24 relative).  A clipped value carries the factor's rounding to f32,
the product's in f32 and the output's: 2 x 2^-24 plus half a step of a 16-bit output, and half the smallest subnormal."""
import pytest
import torch

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
HALF = {F32: 0.0, BF16: 2.0 ** -8, F16: 2.0 ** -11}
TINY = {F32: 2.0 ** -150, BF16: 2.0 ** -134, F16: 2.0 ** -25}


def _norm(ts):
    return sum((t.double() ** 2).sum() for t in ts).sqrt().item()


def _check_norm(got, want):
    assert got.dtype == F32 and got.dim() == 0
    assert abs(got.double().item() - want) <= 2.0 ** -24 * (1 + 1e-6) * want


def _check_clip(outs, ts, want_norm, max_norm):
    scale = min(1.0, max_norm / (want_norm + 1e-6))
    for o, t in zip(outs, ts):
        ref = t.double() * scale
        tol = ref.abs() * (2 * 2.0 ** -24 + HALF[o.dtype]) * (1 + 1e-3) + TINY[o.dtype]
        assert bool(((o.double() - ref).abs() <= tol).all()), (o.dtype, tuple(t.shape))


SIZES = [[1], [2047], [2048], [2049], [65, 1, 128, 147456, 2], [8191, 8193, 16385], [3_000_017], [17_000_003, 5], [7] * 300, [1000 + 37 * i for i in range(131)], [4095, 4096, 4097] * 100]


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("sizes", SIZES)
def test_norm_and_clip_match_the_formula(sizes, dtype):
    from muzero_amd.gradnorm import clip_grad_norm, grad_norm
    g = torch.Generator(device="cuda").manual_seed(len(sizes) + sizes[0])
    ts = [(torch.randn(s, device="cuda", generator=g) * 10.0 ** -(i % 3)).to(dtype) for i, s in enumerate(sizes)]
    want = _norm(ts)
    first = grad_norm(ts)
    _check_norm(first, want)
    assert torch.equal(grad_norm(ts), first)                    # a fixed order: the same bits
    for max_norm in (0.5 * want, 3.0 * want):
        for out_dtype in {dtype, F32}:
            outs = [torch.full(t.shape, 7.0, dtype=out_dtype, device="cuda") for t in ts]
            assert torch.equal(clip_grad_norm(ts, max_norm, out=outs), first)
            _check_clip(outs, ts, want, max_norm)
        mine = [t.clone() for t in ts]
        assert torch.equal(clip_grad_norm(mine, max_norm), first)
        _check_clip(mine, ts, want, max_norm)
        if max_norm > want:
            assert all(torch.equal(a, b) for a, b in zip(mine, ts))   # not clipped: as they were


def test_large_lists_take_the_wide_chunks():
    from muzero_amd.gradnorm import clip_grad_norm, grad_norm
    g = torch.Generator(device="cuda").manual_seed(3)
    ts = [torch.randn(s, device="cuda", generator=g).to(d) for s, d in ((33_000_001, BF16), (9, F32), (20_000_003, F32), (16385, F16))]
    want = _norm(ts)
    _check_norm(grad_norm(ts), want)
    outs = [torch.empty(t.shape, dtype=F32, device="cuda") for t in ts]
    _check_norm(clip_grad_norm(ts, 1.0, out=outs), want)
    _check_clip(outs, ts, want, 1.0)
    mine = [t.clone() for t in ts]
    clip_grad_norm(mine, 1.0)
    _check_clip(mine, ts, want, 1.0)


def test_mixed_types_views_orders_and_empty_tensors():
    from muzero_amd.gradnorm import clip_grad_norm, grad_norm
    g = torch.Generator(device="cuda").manual_seed(4)
    flat = torch.randn(20_001, device="cuda", generator=g)
    half = torch.randn(5_003, device="cuda", generator=g).to(BF16)
    conv = torch.randn(64, 16, 3, 3, device="cuda", generator=g).to(memory_format=torch.channels_last)
    before = [flat.clone(), half.clone(), conv.clone()]
    ts = [flat[1:8194], half[3:5001], conv, torch.empty(0, device="cuda"), torch.randn(33, device="cuda", generator=g).to(F16).t(), torch.randn(7, 9, device="cuda", generator=g).t()]
    kept = [t.clone() for t in ts]
    want = _norm(ts)
    _check_norm(grad_norm(ts), want)
    _check_norm(clip_grad_norm(ts, 2.0), want)
    _check_clip(ts, kept, want, 2.0)
    assert torch.equal(flat[:1], before[0][:1]) and torch.equal(flat[8194:], before[0][8194:])      # what lies beside a view stays
    assert torch.equal(half[:3], before[1][:3]) and torch.equal(half[5001:], before[1][5001:])
    _check_norm(grad_norm(flat), _norm([flat]))                                                    # a tensor is a list of one
    empty = [torch.empty(0, device="cuda"), torch.empty((0, 3), device="cuda")]
    assert grad_norm(empty).item() == 0.0 and clip_grad_norm(empty, 1.0).item() == 0.0


def test_extreme_values_follow_the_formula():
    from muzero_amd.gradnorm import clip_grad_norm, grad_norm
    big = torch.full((1000,), 1e30, device="cuda")
    _check_norm(grad_norm(big), _norm([big]))                   # its squares overflow f32
    small = torch.full((1000,), 1e-30, device="cuda")
    _check_norm(grad_norm(small), _norm([small]))               # its squares underflow f32
    zero = torch.zeros(1000, device="cuda")
    assert clip_grad_norm(zero, 1.0).item() == 0.0 and torch.equal(zero, torch.zeros_like(zero))
    t = torch.tensor([1.0, float("inf"), -2.0], device="cuda")
    assert clip_grad_norm(t, 1.0).item() == float("inf")
    assert t[0].item() == 0.0 and t[2].item() == 0.0 and bool(t[1].isnan())
    t = torch.tensor([1.0, float("nan"), -2.0], device="cuda")
    assert bool(clip_grad_norm(t, 1.0).isnan()) and bool(t.isnan().all())
    t = torch.ones(8, device="cuda")
    clip_grad_norm(t, 0.0)
    assert torch.equal(t, torch.zeros_like(t))
    t = torch.ones(8, device="cuda")
    clip_grad_norm(t, float("inf"))
    assert torch.equal(t, torch.ones_like(t))


def test_two_streams_at_once_and_replayed_graphs():
    from muzero_amd.gradnorm import clip_grad_norm, grad_norm
    g = torch.Generator(device="cuda").manual_seed(6)
    ts = [torch.randn(s, device="cuda", generator=g) for s in (100_003, 17, 4_000_001)]
    us = [torch.randn(s, device="cuda", generator=g) for s in (3_000_001, 77)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = []
    for _ in range(3):
        for st, x in zip(streams, (ts, us)):
            with torch.cuda.stream(st):
                got.append((grad_norm(x), x))
    torch.cuda.synchronize()
    for n, x in got:
        _check_norm(n, _norm(x))
    out = [torch.empty_like(t) for t in ts]
    clip_grad_norm(ts, 1.0, out=out)
    torch.cuda.synchronize()
    graphs = []
    for x in (ts, us):
        o = [torch.empty_like(t) for t in x]
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            n = clip_grad_norm(x, 1.0, out=o)
        graphs.append((gr, x, o, n))
    for k in range(3):
        for _, x, _, _ in graphs:
            for t in x:
                t.mul_(1.5)
        for gr, *_ in graphs:
            gr.replay()
        torch.cuda.synchronize()
        for _, x, o, n in graphs:
            want = _norm(x)
            _check_norm(n, want)
            _check_clip(o, x, want, 1.0)
            assert torch.equal(n, grad_norm(x))


def test_autograd_notices_what_was_scaled():
    from muzero_amd.gradnorm import clip_grad_norm
    x = torch.ones(64, device="cuda", requires_grad=True)
    y = x * 2.0
    z = (y * y).sum()                                    # keeps y
    clip_grad_norm(y, 1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        z.backward()


def test_refusals():
    from muzero_amd import _lib as L
    from muzero_amd.gradnorm import clip_grad_norm, grad_norm
    t = torch.ones(64, device="cuda")
    for bad in ([t, torch.zeros(3)], [t.double()], [t.view(8, 8)[:, ::2]], [t[:1].expand(5)], []):
        with pytest.raises(L.MzError):
            grad_norm(bad)
        with pytest.raises(L.MzError):
            clip_grad_norm(bad, 1.0)
    for kw in (dict(max_norm=-1.0), dict(max_norm=float("nan")), dict(max_norm=1.0, out=[t.clone(), t.clone()]), dict(max_norm=1.0, out=[t.clone().view(8, 8)]),
               dict(max_norm=1.0, out=[t.to(BF16)]), dict(max_norm=1.0, out=[torch.zeros(64)])):
        with pytest.raises(L.MzError):
            clip_grad_norm([t], **kw)
    with pytest.raises(L.MzError, match="overlaps"):
        clip_grad_norm([t, t], 1.0)
    with pytest.raises(L.MzError, match="overlaps"):
        clip_grad_norm([t[:40], t[30:]], 1.0)
    assert torch.equal(t, torch.ones_like(t))
