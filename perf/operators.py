"""Timed cases of the many-tensor operators of training: gradient norm, clipping, the clipped Adam step, moves of rows.

``own = False``: plain torch.  ``own = True``: this package's entry points
(``gsplat_host.optim.grad_norm`` / ``clip_grads_`` / ``GaussianAdam.step(max_norm=...)``,
``gsplat_host.rows.select_rows`` / ``compact_rows``).
"""
import math
import os
import sys

import torch

own = False

_PACKAGE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "gaussian-splatting-own_amd")

_TYPES = {"f32": (torch.float32,), "f16": (torch.float16,), "bf16": (torch.bfloat16,),
          "mixed": (torch.float32, torch.bfloat16, torch.float16)}
_SIZE = {torch.float32: 4, torch.float16: 2, torch.bfloat16: 2}
_LRS = (0.00016, 0.0025, 0.0025 / 20.0, 0.05, 0.005, 0.001)
_NAMES = ("xyz", "f_dc", "f_rest", "opacity", "scaling", "rotation")
_BETA1, _BETA2, _EPS, _STEPS_BEFORE = 0.9, 0.999, 1e-15, 6999


def listed():
    return [
        # the model of a small test: what counts is how long one call takes
        {"name": "norm_5k", "op": "norm", "gaussians": 5003, "rest": 15, "type": "f32", "p": 2.0},
        # a hot scene's gradients, logged every step
        {"name": "norm_6m", "op": "norm", "gaussians": 6_000_000, "rest": 15, "type": "f32", "p": 2.0},
        # many tensors of unlike sizes and types, back to back in one buffer and so aligned to their elements only
        {"name": "norm_301_ragged_mixed", "op": "norm", "tensors": 301, "total": 40_000_000, "type": "mixed", "p": 2.0},
        # a small scene early in training, when nearly every step is clipped
        {"name": "clip_100k", "op": "clip", "gaussians": 100_000, "rest": 15, "type": "f32", "p": 2.0, "clipped": True},
        # a large one later on: the norm stays under the bound and nothing has to be written
        {"name": "clip_1m_under_the_bound", "op": "clip", "gaussians": 1_000_000, "rest": 15, "type": "f32", "p": 2.0,
         "clipped": False},
        # 16-bit gradients of unlike sizes, clipped where they lie
        {"name": "clip_61_ragged_bf16", "op": "clip", "tensors": 61, "total": 120_000_000, "type": "bf16", "p": 2.0,
         "clipped": True},
        # the clipped step of the small model, latency again
        {"name": "step_5k", "op": "step", "gaussians": 5003, "rest": 15, "type": "f32", "p": 2.0, "clipped": True},
        # a million Gaussians whose gradients were exchanged in 16 bits
        {"name": "step_1m_bf16", "op": "step", "gaussians": 1_000_000, "rest": 15, "type": "bf16", "p": 2.0, "clipped": True},
        # the largest scene's step
        {"name": "step_6m", "op": "step", "gaussians": 6_000_000, "rest": 15, "type": "f32", "p": 2.0, "clipped": True},
        # refinement of the small model: parameters and both moments, eighteen tensors
        {"name": "compact_5k", "op": "compact", "gaussians": 5003, "rest": 15, "appended": 401, "kept": 0.9, "runs": 1},
        # copies and children of the restless tenth of a million Gaussians
        {"name": "select_1m", "op": "select", "gaussians": 1_000_000, "rest": 15, "picked": 100_000, "fresh": 0.0,
         "index": "i64"},
        # refinement of the largest scene, the faint ones scattered among the rest
        {"name": "compact_6m", "op": "compact", "gaussians": 6_000_000, "rest": 15, "appended": 300_000, "kept": 0.9,
         "runs": 1},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("norm", "clip", "step", "compact", "select"))
    rest = rng.choice((15, 15, 8, 3, 0))
    if op == "compact":
        n = _log_int(rng, 50, 5_000_000)
        return {"op": op, "gaussians": n, "rest": rest, "appended": rng.choice((0, n // 50, n // 7)),
                "kept": round(rng.uniform(0.3, 1.0), 2), "runs": rng.choice((1, 1, 40, 5000))}
    if op == "select":
        n = _log_int(rng, 50, 5_000_000)
        return {"op": op, "gaussians": n, "rest": rest, "picked": max(1, int(n * rng.uniform(0.01, 1.2))),
                "fresh": rng.choice((0.0, 0.0, 0.2)), "index": rng.choice(("i64", "i32"))}
    case = {"op": op}
    if op != "step" and rng.random() < 0.4:
        case.update(tensors=rng.randint(1, 400 if op == "norm" else 60), total=_log_int(rng, 2_000, 100_000_000))
    else:
        case.update(gaussians=_log_int(rng, 50, 5_000_000), rest=rest)
    case["type"] = rng.choice(("f32", "f32", "bf16", "f16") if op == "step" else ("f32", "f32", "bf16", "f16", "mixed"))
    case["p"] = rng.choice((2.0, 2.0, 1.0, math.inf))
    if op != "norm":
        case["clipped"] = rng.random() < 0.7
    return case


def _model_shapes(case):
    n, rest = case["gaussians"], case["rest"]
    return [(n, 3), (n, 1, 3), (n, rest, 3), (n, 1), (n, 3), (n, 4)]


def _counts(case):
    """Elements of each gradient: the model's six, or sizes that spread over three decades and sum to about ``total``."""
    if "gaussians" in case:
        return [math.prod(s) for s in _model_shapes(case)]
    k = case["tensors"]
    weights = [10.0 ** (3.0 * ((i * 0.618034) % 1.0)) for i in range(k)]
    return [max(1, int(case["total"] * w / sum(weights))) | 1 for w in weights]


def _kept(case):
    return int(round(case["kept"] * (case["gaussians"] + case["appended"])))


def _gradients(n, gen, dtype):
    """Heavy tails, and more than half of it zero: most Gaussians of a scene are hidden in any one view."""
    spread = torch.randn(n, generator=gen, device="cuda").mul_(2.0).exp_().mul_(1e-4)
    g = torch.randn(n, generator=gen, device="cuda").mul_(spread)
    seen = torch.rand((n + 58) // 59, generator=gen, device="cuda") < 0.4
    g = g * seen.repeat_interleave(59)[:n]
    return (g * 256.0 if dtype == torch.float16 else g).to(dtype)          # 16-bit floats carry a loss scale


def _norm_of(grads, p):
    if p == math.inf:
        return torch.stack([g.float().abs().amax() if g.numel() else g.new_zeros((), dtype=torch.float32) for g in grads]).amax()
    powers = [(g.float().abs() if p == 1.0 else g.float().square()).sum(dtype=torch.float64) for g in grads]
    total = torch.stack(powers).sum()
    return (total if p == 1.0 else total.sqrt()).float()


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    op = case["op"]
    state = {"op": op}
    if own:
        if _PACKAGE not in sys.path:
            sys.path.insert(0, _PACKAGE)
        from gsplat_host import optim, rows
        state["optim"], state["rows"] = optim, rows
    if op in ("compact", "select"):
        shapes = _model_shapes(case)
        n, tensors = case["gaussians"], 3 if op == "compact" else 1
        state["tensors"] = [torch.randn(s, generator=gen, device="cuda") for _ in range(tensors) for s in shapes]
        if op == "select":
            index = torch.randint(0, n, (case["picked"],), generator=gen, device="cuda").sort().values
            if case["fresh"]:
                index[torch.rand(index.shape, generator=gen, device="cuda") < case["fresh"]] = -1
            state["index"] = index if case["index"] == "i64" else index.to(torch.int32)
            return state
        extra = case["appended"]
        # new rows come with parameters; their moments start at zero
        state["appended"] = [torch.randn((extra,) + s[1:], generator=gen, device="cuda") for s in shapes] + [None] * 12
        order = torch.rand(((n + extra) // case["runs"] + 1,), generator=gen, device="cuda")
        order = order.repeat_interleave(case["runs"])[:n + extra].argsort()
        state["keep"] = torch.zeros((n + extra,), dtype=torch.bool, device="cuda")
        state["keep"][order[:_kept(case)]] = True
        return state
    counts, types = _counts(case), _TYPES[case["type"]]
    state["p"] = case["p"]
    if "gaussians" in case:
        grads = [_gradients(c, gen, types[i % len(types)]).view(s)
                 for i, (c, s) in enumerate(zip(counts, _model_shapes(case)))]
    else:                                       # back to back in one buffer of each type
        own_counts = {t: [c for i, c in enumerate(counts) if types[i % len(types)] == t] for t in types}
        split = {t: iter(_gradients(sum(c), gen, t).split(c)) for t, c in own_counts.items() if c}
        grads = [next(split[types[i % len(types)]]) for i in range(len(counts))]
    state["grads"] = grads
    if op == "norm":
        return state
    norm = float(_norm_of(grads, case["p"]))
    state["clipped"] = case["clipped"]
    state["max_norm"] = norm * (0.37 if case["clipped"] else 1.7) or 1.0
    if op == "step":
        scale = 2.0 ** -8 if case["type"] == "f16" else 0.125             # the loss scale, or one of eight ranks
        state["grad_scale"] = scale
        state["max_norm"] *= scale
        state["params"] = [torch.randn(s, generator=gen, device="cuda") for s in _model_shapes(case)]
        state["exp_avg"] = [_gradients(c, gen, torch.float32).view(s) for c, s in zip(counts, _model_shapes(case))]
        state["exp_avg_sq"] = [m * m * 2.0 + 1e-12 for m in state["exp_avg"]]
        state["step"] = _STEPS_BEFORE
        if own:
            opt = state["optim"].GaussianAdam(dict(zip(_NAMES, state["params"])), dict(zip(_NAMES, _LRS)))
            opt.exp_avg, opt.exp_avg_sq = dict(zip(_NAMES, state["exp_avg"])), dict(zip(_NAMES, state["exp_avg_sq"]))
            opt.step_count = _STEPS_BEFORE
            state["optimizer"], state["named"] = opt, dict(zip(_NAMES, grads))
    return state


def _bound(state):
    """The bound of this pass.  Clipping leaves gradients of just that norm, so the next pass gets one a ten-thousandth
    lower: each pass then has all of its work to do, as with the fresh gradients of a training loop."""
    bound = state["max_norm"]
    if state["clipped"]:
        state["max_norm"] = bound * 0.9999
    return bound


def _coefficient(norm, bound):
    return (bound / (norm + 1e-6)).clamp(max=1.0)


def _plain_step(state):
    grads = state["grads"]
    norm = _norm_of(grads, state["p"]) * state["grad_scale"]
    c = _coefficient(norm, state["max_norm"]) * state["grad_scale"]
    state["step"] += 1
    bc1, bc2 = 1.0 - _BETA1 ** state["step"], 1.0 - _BETA2 ** state["step"]
    scaled = [g.float() * c for g in grads]
    m = [m.add_((g - m) * (1.0 - _BETA1)) for m, g in zip(state["exp_avg"], scaled)]
    v = [v.mul_(_BETA2).add_(g * g * (1.0 - _BETA2)) for v, g in zip(state["exp_avg_sq"], scaled)]
    p = [p.sub_(a / (b.sqrt() / math.sqrt(bc2) + _EPS) * (lr / bc1))
         for p, a, b, lr in zip(state["params"], m, v, _LRS)]
    return {"norm": norm, "params": p, "exp_avg": m, "exp_avg_sq": v}


def _plain_select(t, index):
    inside = (index >= 0) & (index < t.shape[0])
    rows = t[index.long().clamp(0, t.shape[0] - 1)]
    return rows * inside.view((-1,) + (1,) * (t.dim() - 1))


def _plain_compact(t, extra, fresh, keep):
    return torch.cat((t, t.new_zeros((fresh,) + t.shape[1:]) if extra is None else extra))[keep]


def run(state):
    op = state["op"]
    if op == "norm":
        return state["optim"].grad_norm(state["grads"], state["p"]) if own else _norm_of(state["grads"], state["p"])
    if op == "clip":
        bound, grads = _bound(state), state["grads"]
        if own:
            norm = state["optim"].clip_grads_(grads, bound, state["p"])
        else:
            norm = _norm_of(grads, state["p"])
            c = _coefficient(norm, bound)
            grads = [g.copy_(g.float() * c) for g in grads]
        return {"norm": norm, "grads": grads}
    if op == "step":
        if not own:
            return _plain_step(state)
        norm = state["optimizer"].step(state["named"], state["grad_scale"], max_norm=state["max_norm"], norm_type=state["p"])
        return {"norm": norm, "params": state["params"], "exp_avg": state["exp_avg"], "exp_avg_sq": state["exp_avg_sq"]}
    if op == "select":
        if own:
            return state["rows"].select_rows(state["tensors"], state["index"])
        return [_plain_select(t, state["index"]) for t in state["tensors"]]
    if own:
        out, index = state["rows"].compact_rows(state["tensors"], state["keep"], state["appended"])
        return {"rows": out, "index": index}
    keep = state["keep"]
    fresh = keep.numel() - state["tensors"][0].shape[0]
    return {"rows": [_plain_compact(t, a, fresh, keep) for t, a in zip(state["tensors"], state["appended"])],
            "index": keep.nonzero().view(-1).to(torch.int32)}


def work(case):
    op = case["op"]
    if op == "select":
        row = 4 * (14 + 3 * case["rest"])
        inside = 1.0 - case["fresh"]
        return {"bytes": case["picked"] * (row * (1.0 + inside) + (8 if case["index"] == "i64" else 4)), "flops": 0}
    if op == "compact":
        n, extra = case["gaussians"], case["appended"]
        row = 4 * (14 + 3 * case["rest"])
        # appended rows of the moments are zeros: written, not read
        read = (3 * n + extra) * row * _kept(case) / (n + extra)
        return {"bytes": read + _kept(case) * (3 * row + 4) + n + extra, "flops": 0}
    types = _TYPES[case["type"]]
    counts = _counts(case)
    elements = sum(counts)
    size = sum(c * _SIZE[types[i % len(types)]] for i, c in enumerate(counts))
    if op == "norm":
        return {"bytes": size + 4, "flops": 2 * elements}
    if op == "clip":
        return {"bytes": size * (2 if case["clipped"] else 1) + 4, "flops": 3 * elements}
    return {"bytes": size + 24 * elements + 4, "flops": 18 * elements}


def _exact_norm(grads, p):
    flat = torch.cat([g.reshape(-1).to(torch.float64) for g in grads])
    return flat.abs().max() if p == math.inf else flat.abs().sum() if p == 1.0 else torch.dot(flat, flat) ** 0.5


def exact(case, seed):
    state = prepare(case, seed)
    op = case["op"]
    if op == "select":
        index = state["index"].to(torch.int64)
        out = [torch.zeros((index.numel(),) + t.shape[1:], dtype=torch.float64, device="cuda") for t in state["tensors"]]
        at = (index >= 0).nonzero().view(-1)
        return [o.index_copy_(0, at, t.double().index_select(0, index[at])) for o, t in zip(out, state["tensors"])]
    if op == "compact":
        index = torch.arange(state["keep"].numel(), device="cuda").masked_select(state["keep"])
        n = case["gaussians"]
        old, new = index[index < n], index[index >= n] - n
        return {"rows": [torch.cat((t.index_select(0, old), a.index_select(0, new) if a is not None else
                                    t.new_zeros((new.numel(),) + t.shape[1:]))).double()
                         for t, a in zip(state["tensors"], state["appended"])], "index": index.to(torch.int32)}
    norm = _exact_norm(state["grads"], case["p"])
    if op == "norm":
        return norm
    if op == "clip":
        factor = min(1.0, state["max_norm"] / (float(norm) + 1e-6))
        return {"norm": norm, "grads": [g.double() * factor for g in state["grads"]]}
    norm = norm * state["grad_scale"]
    factor = state["grad_scale"] * min(1.0, state["max_norm"] / (float(norm) + 1e-6))
    t = _STEPS_BEFORE + 1
    g = [x.double() * factor for x in state["grads"]]
    m = [_BETA1 * a.double() + (1.0 - _BETA1) * x for a, x in zip(state["exp_avg"], g)]
    v = [_BETA2 * a.double() + (1.0 - _BETA2) * x ** 2 for a, x in zip(state["exp_avg_sq"], g)]
    p = [a.double() - lr * (x / (1.0 - _BETA1 ** t)) / ((y / (1.0 - _BETA2 ** t)) ** 0.5 + _EPS)
         for a, x, y, lr in zip(state["params"], m, v, _LRS)]
    return {"norm": norm, "params": p, "exp_avg": m, "exp_avg_sq": v}
