"""Timed cases of the policy's and the update's operators: sampling an action from logits, the policy's cross-entropy with its
gradient, the global gradient norm and clipping by it.

`own` chooses between the framework's kernels (muzero_amd.policy, muzero_amd.gradnorm) and the same operators written out in
elementary torch operations; `exact` has them in 64 bits, written a second time."""
import math

import torch

own = False

DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}
MOST = 4096 * 32768      # elements of the largest loss case


# ---- the cases ------------------------------------------------------------------------------------------------------------
def _sample(name, n, v, dtype, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, legal="none", rows=False, pad=0):
    return {"name": name, "op": "sample", "n": n, "v": v, "dtype": dtype, "temperature": temperature, "top_k": top_k, "top_p": top_p,
            "min_p": min_p, "legal": legal, "rows": rows, "pad": pad}


def _loss(name, n, v, dtype, target, legal="none", weight=False, pad=0):
    return {"name": name, "op": "loss", "n": n, "v": v, "dtype": dtype, "target": target, "legal": legal, "weight": weight, "pad": pad}


def _norm(name, op, shapes, dtype, count=0, elements=0, out="same", max_norm=1.0):
    return {"name": name, "op": op, "shapes": shapes, "dtype": dtype, "count": count, "elements": elements, "out": out, "max_norm": max_norm}


def listed():
    return [
        # the moves of a handful of games, straight from their policy over 64 squares + pass: latency only
        _sample("moves-8", 8, 65, "f32", legal="board"),
        # one move in each of 4096 lock-step games at the arena's temperature (the batch that the search is run with)
        _sample("moves-4096", 4096, 65, "f32", temperature=0.25, legal="board"),
        # few requests that decode over a large vocabulary, with the usual filters together
        _sample("vocab-4", 4, 131072, "f32", temperature=0.8, top_k=50, top_p=0.9),
        # a serving batch whose requests carry their own settings; odd vocabulary, rows cut from a wider buffer, forbidden tokens
        _sample("vocab-61-ragged", 61, 100003, "bf16", temperature=0.9, top_k=0, top_p=0.95, min_p=0.02, legal="bool", rows=True, pad=5),
        # a full serving batch, nucleus only: the total mass of every row is needed
        _sample("vocab-256", 256, 131072, "bf16", temperature=1.0, top_p=0.9),
        # one training step's policy rows: (3 + 1) unrolled steps of a batch of 512, targets from visit counts
        _loss("policy-2048", 2048, 65, "f32", "f32"),
        # odd sizes in 16 bits: forbidden actions, row weights with padding rows among them, a row without a legal action
        _loss("loss-777-ragged", 777, 5003, "f16", "f32", legal="bool", weight=True, pad=3),
        # few long rows: a distillation step of a single short sequence
        _loss("loss-8", 8, 131072, "f32", "f32"),
        # a large distillation step, everything in 16 bits
        _loss("loss-4096", 4096, 32768, "bf16", "bf16"),
        # this framework's own gradients, tensor by tensor, clipped before the optimiser's step
        _norm("clip-net", "clip", "net", "f32"),
        # the norm alone, over many small and ragged tensors (what a step logs)
        _norm("norm-many", "norm", "ragged", "bf16", count=400, elements=40_000_000),
        # a large model's 16-bit gradients clipped into the 32-bit ones that its optimiser reads
        _norm("clip-large", "clip", "ragged", "bf16", count=24, elements=400_000_000, out="f32"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["sample", "sample", "loss", "loss", "norm", "clip"])
    dtype = rng.choice(["f32", "bf16", "f16"])
    if op == "sample":
        v = 65 if rng.random() < 0.2 else _log(rng, 2, 200_000)
        n = _log(rng, 16 if v < 1000 else 4, min(4096, MOST // 2 // SIZE[dtype] // v))
        c = _sample("", n, v, dtype, temperature=rng.choice([0.0, 0.25, round(rng.uniform(0.3, 1.5), 3), 1.0]), top_k=rng.choice([0, 0, 1, _log(rng, 2, 2000)]),
                    top_p=rng.choice([1.0, round(rng.uniform(0.05, 0.99), 3)]), min_p=rng.choice([0.0, 0.0, round(rng.uniform(0.001, 0.5), 4)]),
                    legal=rng.choice(["none", "bool"] + (["board"] * 2 if v == 65 else [])), rows=rng.random() < 0.3, pad=rng.choice([0, 0, rng.randint(1, 9)]))
    elif op == "loss":
        v = 65 if rng.random() < 0.2 else _log(rng, 2, 200_000)
        n = _log(rng, 16 if v < 1000 else 1, min(16384, MOST // SIZE[dtype] // v))
        c = _loss("", n, v, dtype, rng.choice(["f32", dtype]), legal=rng.choice(["none", "none", "bool"] + (["board"] if v == 65 else [])),
                  weight=rng.random() < 0.4, pad=rng.choice([0, 0, rng.randint(1, 9)]))
    else:
        e = _log(rng, 100, 300_000_000 if dtype == "f32" else 400_000_000)
        c = _norm("", op, "ragged", dtype, count=min(e, _log(rng, 1, 60 if op == "clip" else 600)), elements=e, out=rng.choice(["same", "f32"]),
                  max_norm=rng.choice([0.5, 1.0, 1e9]))
    del c["name"]
    return c


# ---- the inputs -----------------------------------------------------------------------------------------------------------
def _net_shapes():
    """the trainable tensors of the representation, prediction and dynamics networks"""
    tower = [(128, 128, 3, 3), (128,)] * 6
    return ([(128, 9, 3, 3), (128,)] + tower + [(8, 128, 3, 3), (8,)]
            + [(2, 8, 1, 1), (2,), (128, 128), (128,), (65, 128), (65,), (2, 8, 1, 1), (2,), (1, 128), (1,)]
            + [(128, 10, 3, 3)] + tower + [(8, 128, 3, 3)])


def _ragged_sizes(count, elements):
    """sizes that fall off over four powers of ten, odd ones among them, and add up to about `elements`"""
    share = [10.0 ** (-4.0 * ((7 * i) % count) / count) for i in range(count)]
    return [max(1, int(elements * s / sum(share))) | 1 for s in share]


def _shapes(case):
    return _net_shapes() if case["shapes"] == "net" else [(s,) for s in _ragged_sizes(case["count"], case["elements"])]


def _cut(t, pad):
    """the same values as rows of a wider buffer, from its second column on"""
    if not pad:
        return t
    wide = torch.zeros((t.shape[0], t.shape[1] + pad), dtype=t.dtype, device=t.device)
    wide[:, 1:1 + t.shape[1]] = t
    return wide[:, 1:1 + t.shape[1]]


def _mask(case, gen):
    n, v = case["n"], case["v"]
    if case["legal"] == "none":
        return None
    if case["legal"] == "board":   # a mover's placements as a bitboard: about ten squares, now and then none (the pass)
        bits = torch.rand((n, 64), device="cuda", generator=gen) < 0.15
        bits[5::17] = False
        shift = torch.arange(64, device="cuda")
        return (bits.long() << shift).sum(1)
    m = torch.rand((n, v), device="cuda", generator=gen) < 0.8
    if n > 2:
        m[1] = False               # a row that its mask leaves empty
    return m


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed) * 7919 + 13)
    rand = lambda *s: torch.rand(s, device="cuda", generator=gen)      # noqa: E731
    randn = lambda *s: torch.randn(s, device="cuda", generator=gen)    # noqa: E731
    s = {"case": case}
    if case["op"] in ("norm", "clip"):
        shapes = _shapes(case)
        s["grads"] = [(randn(*sh) * 10.0 ** float(-1 - i % 4)).to(DT[case["dtype"]]) for i, sh in enumerate(shapes)]
        if case["op"] == "clip":
            s["out"] = [torch.empty(sh, dtype=DT[case["dtype"] if case["out"] == "same" else "f32"], device="cuda") for sh in shapes]
        return s
    n, v = case["n"], case["v"]
    x = randn(n, v)
    x = 2.0 * x + 6.0 * (x - 2.0).clamp_(min=0.0) if v > 256 else 1.5 * x     # a bulk with a few that stand out
    s["legal"] = _mask(case, gen)
    if case["op"] == "sample":
        s["logits"] = _cut(x.to(DT[case["dtype"]]), case["pad"])
        s["u"] = torch.rand(n, dtype=torch.float64, device="cuda", generator=gen)
        s["set"] = {k: case[k] for k in ("temperature", "top_k", "top_p", "min_p")}
        if case["rows"]:           # every request with settings of its own around these; some greedy, some without a filter
            some = rand(n)
            s["set"] = {"temperature": torch.where(some < 0.1, 0.0, case["temperature"] * (0.5 + rand(n))),
                        "top_k": torch.where(some > 0.7, torch.randint(1, 100, (n,), device="cuda", generator=gen), case["top_k"]).to(torch.int32),
                        "top_p": torch.where(some > 0.9, 1.0, case["top_p"] * (0.8 + 0.2 * rand(n))),
                        "min_p": case["min_p"] * rand(n)}
        return s
    t = randn(n, v).mul_(2.0).softmax(1)      # visit shares, or another model's probabilities
    if case["legal"] == "bool":
        t *= s["legal"]
        t /= t.sum(1, keepdim=True).clamp(min=1e-30)
    s["targets"] = t.to(DT[case["target"]])
    s["logits"] = _cut(x.to(DT[case["dtype"]]), case["pad"]).detach().requires_grad_()
    s["weight"] = None
    if case["weight"]:
        s["weight"] = 0.5 + rand(n)
        s["weight"][3::5] = 0.0                # padding rows
    return s


# ---- the plain forms --------------------------------------------------------------------------------------------------------
def _allowed(legal, v):
    """(n, v) truth values of what may be played: given as they are, or 64 squares of a bitboard and the pass where none is free"""
    if legal is None or legal.dim() == 2:
        return legal
    squares = ((legal.unsqueeze(1) >> torch.arange(64, device=legal.device)) & 1) != 0
    return torch.cat((squares, (legal == 0).unsqueeze(1)), dim=1)


def _column(p, like):
    return p.to(like.dtype).unsqueeze(1) if torch.is_tensor(p) else torch.full((like.shape[0], 1), float(p), dtype=like.dtype, device=like.device)


def _plain_sample(logits, u, legal, temperature, top_k, top_p, min_p):
    """in 64 bits: a draw next to the border of two actions has to fall on the same side"""
    x = logits.double()
    allowed = _allowed(legal, x.shape[1])
    if allowed is not None:
        x = x.masked_fill(~allowed, -math.inf)
    x, order = torch.sort(x, dim=1, descending=True, stable=True)
    temperature, top_k, top_p, min_p = (_column(p, x) for p in (temperature, top_k, top_p, min_p))
    w = torch.exp((x - x[:, :1]) / torch.where(temperature > 0, temperature, torch.ones_like(temperature)))
    place = torch.arange(x.shape[1], device=x.device)
    in_k = (place < top_k) | (top_k <= 0)
    kw = w * in_k
    before = torch.cumsum(kw, 1) - kw
    keep = in_k & ((before < top_p * kw.sum(1, keepdim=True)) | (top_p >= 1)) & (w >= min_p)
    keep[:, 0] = True
    keep = keep & ((temperature > 0) | (place == 0))
    mass = torch.zeros_like(w).scatter_(1, order, w * keep)       # back into the actions' own order
    cum = torch.cumsum(mass, 1)
    pick = (cum > u.unsqueeze(1) * cum[:, -1:]).int().argmax(1)   # the first
    return torch.where(x[:, 0] > -math.inf, pick, -1).int()


def _plain_loss(logits, targets, weight, legal):
    x, t = logits.detach().float(), targets.float()
    allowed = _allowed(legal, x.shape[1])
    if allowed is not None:
        x = x.masked_fill(~allowed, -math.inf)
        t = t.masked_fill(~allowed, 0.0)
    m = x.amax(1, keepdim=True)
    some = m > -math.inf
    e = torch.exp(torch.where(some, x - m, -math.inf))
    z = e.sum(1, keepdim=True)
    ts = t.sum(1, keepdim=True)
    row = ts * torch.log(z) - (t * torch.where(t != 0, x - m, 0.0)).sum(1, keepdim=True)
    scale = (torch.ones_like(m) if weight is None else weight.unsqueeze(1)) * some / x.shape[0]
    loss = torch.where(scale != 0, row * scale, 0.0).sum(dtype=torch.float64).float()
    grad = torch.where(scale != 0, (e / z * ts - t) * scale, 0.0)
    return [loss, grad.to(logits.dtype)]


def _plain_norm(grads):
    return torch.stack([g.float().square().sum(dtype=torch.float64) for g in grads]).sum().sqrt().float()


def run(state):
    case = state["case"]
    if case["op"] == "sample":
        if own:
            from muzero_amd import policy
            return policy.sample_actions(state["logits"], state["u"], legal=state["legal"], **state["set"])
        return _plain_sample(state["logits"], state["u"], state["legal"], **state["set"])
    if case["op"] == "loss":
        if own:
            from muzero_amd import policy
            loss = policy.cross_entropy(state["logits"], state["targets"], weight=state["weight"], legal=state["legal"])
            return [loss.detach(), torch.autograd.grad(loss, state["logits"])[0]]
        return _plain_loss(state["logits"], state["targets"], state["weight"], state["legal"])
    if case["op"] == "norm":
        if own:
            from muzero_amd import gradnorm
            return gradnorm.grad_norm(state["grads"])
        return _plain_norm(state["grads"])
    if own:
        from muzero_amd import gradnorm
        return [gradnorm.clip_grad_norm(state["grads"], case["max_norm"], out=state["out"])] + state["out"]
    norm = _plain_norm(state["grads"])
    scale = (case["max_norm"] / (norm + 1e-6)).clamp(max=1.0)
    return [norm] + [o.copy_(g.float() * scale) for g, o in zip(state["grads"], state["out"])]


# ---- what a pass cannot do without -------------------------------------------------------------------------------------------
def work(case):
    if case["op"] in ("norm", "clip"):
        e = sum(math.prod(s) for s in _shapes(case))
        out = SIZE[case["dtype"] if case["out"] == "same" else "f32"] if case["op"] == "clip" else 0
        return {"bytes": e * (SIZE[case["dtype"]] + out) + 4, "flops": e * (3 if out else 2)}
    n, v = case["n"], case["v"]
    mask = {"none": 0, "board": 8 * n, "bool": n * v}[case["legal"]]
    if case["op"] == "sample":
        return {"bytes": n * v * SIZE[case["dtype"]] + mask + n * (12 + (16 if case["rows"] else 0)), "flops": 3 * n * v}
    return {"bytes": n * v * (2 * SIZE[case["dtype"]] + SIZE[case["target"]]) + mask + (4 * n if case["weight"] else 0) + 4, "flops": 10 * n * v}


# ---- the definitions in 64 bits ------------------------------------------------------------------------------------------------
def exact(case, seed):
    if case["op"] == "sample":
        return None if case["n"] * case["v"] > 10_000_000 else _exact_sample(prepare(case, seed))
    return _exact_loss(prepare(case, seed)) if case["op"] == "loss" else _exact_norm(prepare(case, seed))


def _exact_sample(s):
    import numpy as np
    x = s["logits"].double().cpu().numpy()
    n, v = x.shape
    allowed = np.ones((n, v), bool)
    if s["legal"] is not None and s["legal"].dim() == 2:
        allowed = s["legal"].cpu().numpy()
    elif s["legal"] is not None:
        for i, board in enumerate(s["legal"].tolist()):
            allowed[i] = [bool(board >> a & 1) for a in range(64)] + [board == 0]
    u = s["u"].cpu().numpy()
    per = [p.double().cpu().tolist() if torch.is_tensor(p) else [p] * n for p in (s["set"][k] for k in ("temperature", "top_k", "top_p", "min_p"))]
    picks = np.full(n, -1, np.int32)
    for i, (temperature, top_k, top_p, min_p) in enumerate(zip(*per)):
        free = np.flatnonzero(allowed[i] & (x[i] > -np.inf))
        if not free.size:
            continue
        free = free[np.argsort(-x[i, free], kind="stable")]       # best first, the lower index of equals first
        if temperature <= 0:
            picks[i] = free[0]
            continue
        if top_k > 0:
            free = free[:int(top_k)]
        p = np.exp((x[i, free] - x[i, free[0]]) / temperature)
        last = free.size
        if top_p < 1:
            last = max(1, int(np.searchsorted(np.concatenate(([0.0], np.cumsum(p)[:-1])), top_p * p.sum(), side="left")))
        last = max(1, min(last, int((p >= min_p).sum())))
        kept = np.sort(free[:last])
        q = np.cumsum(np.exp((x[i, kept] - x[i, free[0]]) / temperature))
        picks[i] = kept[min(int(np.searchsorted(q, u[i] * q[-1], side="right")), kept.size - 1)]
    return torch.from_numpy(picks)


def _exact_loss(s):
    logits, targets, legal, weight = s["logits"].detach(), s["targets"], s["legal"], s["weight"]
    n, v = logits.shape
    grad = torch.zeros((n, v), dtype=torch.float64, device="cuda")
    rows = torch.zeros(n, dtype=torch.float64, device="cuda")
    for a in range(0, n, 512):
        b = min(n, a + 512)
        x, t = logits[a:b].double(), targets[a:b].double()
        if legal is not None:
            ok = legal[a:b] if legal.dim() == 2 else torch.stack([legal[a:b] >> i & 1 for i in range(64)] + [(legal[a:b] == 0).long()], 1).bool()
            x, t = torch.where(ok, x, -math.inf), torch.where(ok, t, 0.0)
        live = torch.isfinite(x.max(1).values)
        w = torch.full((b - a,), 1.0 / n, dtype=torch.float64, device="cuda") if weight is None else weight[a:b].double() / n
        logp = torch.log_softmax(torch.where(live[:, None], x, 0.0), 1)
        rows[a:b] = -w * (t * torch.where(t > 0, logp, 0.0)).sum(1) * live
        grad[a:b] = (logp.exp() * t.sum(1, keepdim=True) - t) * (w * live)[:, None]
    return [rows.sum(), grad]


def _exact_norm(s):
    total = sum(torch.linalg.vector_norm(g.double()).square() for g in s["grads"])
    if s["case"]["op"] == "norm":
        return total.sqrt()
    scale = torch.clamp(s["case"]["max_norm"] / (total.sqrt() + 1e-6), max=1.0)
    return [total.sqrt()] + [(g.double() * scale).reshape(o.shape) for g, o in zip(s["grads"], s["out"])]
