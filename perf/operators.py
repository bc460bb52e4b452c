"""Cases, plain forms and exact values of the row operators: ``povs.sample``, ``povs.route``,
``povs.plan_rows`` with ``povs.dispatch_rows``, and ``povs.combine_rows``.

The plain forms are elementary torch operations.  Scores and weights whose order or running sum
decides a whole number (which expert, which id) are computed in 64 bits, since two of them can lie
closer together than 32 bits tell apart; values that are only returned are rounded once at the end.
"""

from __future__ import annotations

import math
import sys
from pathlib import Path

import torch

own = False

_PACKAGE = str(Path(__file__).resolve().parent.parent / "pov-shuffle_b200")
_DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}


def _povs():
    if _PACKAGE not in sys.path:
        sys.path.insert(0, _PACKAGE)
    import povs

    return povs


def listed():
    return [
        # One answer being written: a single row of scores over an odd vocabulary; latency counts.
        dict(name="sample_one", op="sample", rows=1, width=50021, dtype="float32", temperature=0.8, top_k=40,
             top_p=0.95, min_p=0.0, per_row=False),
        # A serving batch whose requests each bring their own temperature, top-k, top-p and min-p.
        dict(name="sample_mixed_batch", op="sample", rows=96, width=128000, dtype="bfloat16", temperature=1.0,
             top_k=0, top_p=1.0, min_p=0.0, per_row=True),
        # Many sequences drawn at once by nucleus only, the largest scores that a decode step holds.
        dict(name="sample_nucleus_large", op="sample", rows=512, width=131072, dtype="float32", temperature=1.0,
             top_k=0, top_p=0.9, min_p=0.0, per_row=False),
        # A decode step: a few rows routed; latency counts.
        dict(name="route_decode", op="route", rows=13, experts=64, k=6, dtype="bfloat16", scoring="softmax", bias=False,
             groups=1, top_groups=1, renormalize=True, scale=1.0, train=False),
        # A prompt batch: sigmoid scores with a balance bias, experts in groups, weights renormalised and scaled.
        dict(name="route_groups_prompt", op="route", rows=65536, experts=256, k=8, dtype="float32", scoring="sigmoid",
             bias=True, groups=8, top_groups=4, renormalize=True, scale=2.5, train=False),
        # A training step of an odd batch: weights and the gradient of the scores.
        dict(name="route_train", op="route", rows=32749, experts=128, k=8, dtype="bfloat16", scoring="softmax",
             bias=False, groups=1, top_groups=1, renormalize=False, scale=1.0, train=True),
        # A decode step's rows to their experts.
        dict(name="dispatch_decode", op="dispatch", rows=13, experts=64, k=6, width=2048, dtype="bfloat16",
             padding=0.0, train=False),
        # A prompt batch's rows to their experts: the largest move.
        dict(name="dispatch_prompt", op="dispatch", rows=16384, experts=256, k=8, width=4096, dtype="bfloat16",
             padding=0.0, train=False),
        # A padded training batch in 32 bits with an odd row width, and the rows' gradient.
        dict(name="dispatch_train_odd", op="dispatch", rows=8191, experts=60, k=4, width=1023, dtype="float32",
             padding=0.03, train=True),
        # A decode step's expert rows back to its rows.
        dict(name="combine_decode", op="combine", rows=13, experts=64, k=6, width=2048, dtype="bfloat16",
             padding=0.0, train=False),
        # A prompt batch back from its experts.
        dict(name="combine_prompt", op="combine", rows=16384, experts=256, k=8, width=4096, dtype="bfloat16",
             padding=0.0, train=False),
        # A padded training batch: the combined rows, the gradients of the experts' rows and of the weights.
        dict(name="combine_train", op="combine", rows=8191, experts=128, k=6, width=2048, dtype="float16",
             padding=0.03, train=True),
    ]


def _spread(rng, low, high):
    """A whole number spread over the logarithm of low..high."""
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["sample", "route", "dispatch", "combine"])
    dtype = rng.choice(["float32", "bfloat16", "float16"])
    if op == "sample":
        width = _spread(rng, 1000, 262144)
        rows = min(_spread(rng, 1, 512), max(1, 512 * 131072 // width))
        mode = rng.choice(["plain", "top_k", "top_p", "min_p", "all", "per_row"])
        return dict(op=op, rows=rows, width=width, dtype=dtype, temperature=round(rng.uniform(0.6, 1.3), 3),
                    top_k=_spread(rng, 1, 1000) if mode in ("top_k", "all") else 0,
                    top_p=round(rng.uniform(0.5, 0.99), 3) if mode in ("top_p", "all") else 1.0,
                    min_p=round(rng.uniform(0.01, 0.2), 3) if mode in ("min_p", "all") else 0.0,
                    per_row=mode == "per_row")
    if op == "route":
        groups = rng.choice([1, 1, 4, 8])
        experts = groups * max(2, _spread(rng, 8, 512) // groups)
        top_groups = 1 if groups == 1 else rng.randint(max(1, groups // 2), groups)
        k = min(_spread(rng, 1, 12), top_groups * (experts // groups))
        rows = min(_spread(rng, 1, 65536), 65536 * 256 // experts)
        return dict(op=op, rows=rows, experts=experts, k=k, dtype=dtype, scoring=rng.choice(["softmax", "sigmoid"]),
                    bias=rng.random() < 0.5, groups=groups, top_groups=top_groups,
                    renormalize=k > 1 and rng.random() < 0.5,  # one renormalised weight is always 1
                    scale=rng.choice([1.0, 2.5]), train=rng.random() < 0.4)
    train = rng.random() < 0.4
    experts, k = _spread(rng, 8, 512), rng.randint(1, 8)
    width = _spread(rng, 64, 8192)
    if rng.random() < 0.7:  # widths are mostly whole 16-byte pieces
        width = width // 8 * 8
    most = 16384 * 8 * 4096 * 2 // ((8 if train else 1) * k * width * (4 if dtype == "float32" else 2))
    return dict(op=op, rows=min(_spread(rng, 1, 16384), max(1, most)), experts=experts, k=k, width=width, dtype=dtype,
                padding=rng.choice([0.0, 0.0, 0.05]), train=train)


# ------------------------------------------------------------------------------------------
# Inputs.
# ------------------------------------------------------------------------------------------


def _choices(case, g):
    """Distinct experts of each row, some experts more in demand than others; padding rows hold -1."""
    demand = torch.randn(case["experts"], device="cuda", generator=g) * 0.5
    noise = -torch.log(-torch.log(torch.rand(case["rows"], case["experts"], device="cuda", generator=g).clamp_(1e-7, 1 - 1e-7)))
    experts = (demand + noise).topk(min(case["k"], case["experts"]), dim=1).indices.to(torch.int32)
    if case["padding"] > 0:
        experts[torch.rand(case["rows"], device="cuda", generator=g) < case["padding"]] = -1
    return experts


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype = _DTYPES[case["dtype"]]
    rows = case["rows"]
    state = dict(case=case)
    if case["op"] == "sample":
        # Exponentially distributed scores: probabilities fall with a power of the rank, as words' do.
        tail = 1.0 + torch.rand(rows, 1, device="cuda", generator=g)
        noise = torch.rand(rows, case["width"], device="cuda", generator=g).clamp_(1e-7, 1.0)
        logits = noise.log_().mul_(-tail)
        banned = torch.rand(case["width"], device="cuda", generator=g) < 0.01
        logits = logits.masked_fill_(banned, float("-inf")).to(dtype)
        del noise
        state.update(logits=logits, uniforms=torch.rand(rows, device="cuda", generator=g))
        if case["per_row"]:
            pick = torch.randint(0, 5, (4, rows), device="cuda", generator=g)
            state.update(
                temperature=torch.tensor([0.0, 0.6, 0.8, 1.0, 1.2], device="cuda")[pick[0]],
                top_k=torch.tensor([0, 1, 20, 50, 200], device="cuda", dtype=torch.int32)[pick[1]],
                top_p=torch.tensor([1.0, 0.8, 0.9, 0.95, 1.0], device="cuda")[pick[2]],
                min_p=torch.tensor([0.0, 0.0, 0.0, 0.02, 0.1], device="cuda")[pick[3]])
        else:
            state.update({name: case[name] for name in ("temperature", "top_k", "top_p", "min_p")})
        return state
    if case["op"] == "route":
        state["logits"] = (torch.randn(rows, case["experts"], device="cuda", generator=g) * 1.5).to(dtype)
        state["bias"] = torch.randn(case["experts"], device="cuda", generator=g) * 0.05 if case["bias"] else None
        state["grad"] = torch.randn(rows, case["k"], device="cuda", generator=g) if case["train"] else None
        return state
    state["experts"] = experts = _choices(case, g)
    k = experts.shape[1]
    if case["op"] == "dispatch":
        state["data"] = torch.randn(rows, case["width"], device="cuda", generator=g).to(dtype)
        if case["train"]:
            state["grad"] = torch.randn(rows * k, case["width"], device="cuda", generator=g).to(dtype)
        return state
    state["data"] = torch.randn(rows * k, case["width"], device="cuda", generator=g).to(dtype)
    state["weights"] = torch.rand(rows, k, device="cuda", generator=g)
    state["plan"] = _plan(experts, case["experts"])  # what the dispatch before it left in hand
    if case["train"]:
        state["grad"] = torch.randn(rows, case["width"], device="cuda", generator=g).to(dtype)
    return state


# ------------------------------------------------------------------------------------------
# Plain forms.
# ------------------------------------------------------------------------------------------


def _column(value, rows, dtype):
    if isinstance(value, torch.Tensor):
        return value.to(dtype).reshape(rows, 1)
    return torch.full((rows, 1), value, dtype=dtype, device="cuda")


def _sample(state):
    logits, rows = state["logits"].double(), state["case"]["rows"]
    width = logits.shape[1]
    temperature = _column(state["temperature"], rows, torch.float64)
    greedy = temperature <= 0
    ordered, order = logits.sort(dim=1, descending=True, stable=True)  # equal scores: lowest index first
    weight = torch.exp((ordered - ordered[:, :1]) / torch.where(greedy, 1.0, temperature))
    place = torch.arange(width, device="cuda").expand(rows, width)
    top_k = _column(state["top_k"], rows, torch.int64)
    keep = (place < top_k) | (top_k <= 0)
    weight = torch.where(keep, weight, 0.0)
    top_p = _column(state["top_p"], rows, torch.float64)
    running = weight.cumsum(1)
    keep &= (running - weight < top_p * running[:, -1:]) | (top_p >= 1) | (place == 0)
    keep &= weight >= _column(state["min_p"], rows, torch.float64)
    keep &= ~greedy | (place == 0)
    weight = torch.zeros_like(weight).scatter_(1, order, torch.where(keep, weight, 0.0))
    running = weight.cumsum(1)
    target = state["uniforms"].double().reshape(rows, 1) * running[:, -1:]
    return (running <= target).sum(1)


def _best(score, count):
    """Places of the `count` largest of the last dimension, equal ones by the lowest place."""
    return score.argsort(dim=-1, descending=True, stable=True)[..., :count]


def _route(state):
    case, logits, bias, k = state["case"], state["logits"].double(), state["bias"], state["case"]["k"]
    rows, n = logits.shape
    if case["scoring"] == "softmax":
        score = torch.exp(logits - logits.amax(1, keepdim=True))
        score = score / score.sum(1, keepdim=True)
    else:
        score = 1 / (1 + torch.exp(-logits))
    choice = score if bias is None else score + bias.double()
    if case["groups"] > 1:
        grouped = choice.reshape(rows, case["groups"], -1)
        two = grouped.gather(2, _best(grouped, 2))
        kept = torch.zeros(rows, case["groups"], dtype=torch.bool, device="cuda")
        kept.scatter_(1, _best(two.sum(2), case["top_groups"]), True)
        choice = torch.where(kept.unsqueeze(2), grouped, float("-inf")).reshape(rows, n)
    experts = _best(choice, k)
    chosen = score.gather(1, experts)
    total = chosen.sum(1, keepdim=True) if case["renormalize"] else torch.ones_like(chosen[:, :1])
    weights = chosen / total * case["scale"]
    out = [experts.to(torch.int32), weights.float()]
    if case["train"]:
        grad = state["grad"].double() * case["scale"] / total
        if case["renormalize"]:  # d(s_j / S) = (ds_j - (s_j / S) sum of ds) / S
            grad = grad - (grad * chosen / total).sum(1, keepdim=True)
        spread = torch.zeros_like(score).scatter_(1, experts, grad)
        if case["scoring"] == "softmax":
            spread = score * (spread - (grad * chosen).sum(1, keepdim=True))
        else:
            spread = score * (1 - score) * spread
        out.append(spread.to(state["logits"].dtype))
    return out


def _plan(experts, n_experts):
    flat = experts.reshape(-1).long()
    key = torch.where(flat < 0, n_experts, flat)
    order = key.argsort(stable=True)
    valid = (key[order] < n_experts)
    place = torch.arange(flat.numel(), device="cuda")
    slots = torch.empty_like(place).scatter_(0, order, torch.where(valid, place, -1))
    counts = torch.zeros(n_experts + 1, dtype=torch.int64, device="cuda").index_add_(0, key, torch.ones_like(key))
    offsets = torch.cat([counts.new_zeros(1), counts[:n_experts].cumsum(0)])
    return (slots.reshape(experts.shape).to(torch.int32), torch.where(valid, order, -1).to(torch.int32),
            offsets.to(torch.int32))


def _gathered(data, slots):
    """(rows, k, width) in 32 bits: the slots' rows, zeros where a slot is -1."""
    got = data.float()[slots.clamp(min=0).long()]
    return torch.where((slots >= 0).unsqueeze(-1), got, 0.0)


def _dispatch(state):
    case, data = state["case"], state["data"]
    slots, sources, offsets = plan = _plan(state["experts"], case["experts"])
    k = slots.shape[1]
    rows = torch.where((sources >= 0).unsqueeze(1), data[(sources.clamp(min=0) // k).long()], 0)
    out = [rows, *plan]
    if case["train"]:
        out.append(_gathered(state["grad"], slots).sum(1).to(data.dtype))
    return out


def _combine(state):
    data, weights = state["data"], state["weights"]
    slots, sources, _ = state["plan"]
    k = slots.shape[1]
    got = _gathered(data, slots)
    out = [(got * weights.unsqueeze(-1)).sum(1).to(data.dtype)]
    if state["case"]["train"]:
        grad = state["grad"].float()
        at = sources.clamp(min=0).long()
        spread = torch.where((sources >= 0).unsqueeze(1), grad[at // k] * weights.reshape(-1)[at].unsqueeze(1), 0.0)
        out += [spread.to(data.dtype), (got * grad.unsqueeze(1)).sum(2)]
    return out


def _own_run(state):
    povs, case = _povs(), state["case"]
    if case["op"] == "sample":
        return povs.sample(state["logits"], state["uniforms"], temperature=state["temperature"],
                           top_k=state["top_k"], top_p=state["top_p"], min_p=state["min_p"])
    train = case["train"]
    if case["op"] == "route":
        logits = state["logits"].detach().requires_grad_(train)
        experts, weights = povs.route(logits, case["k"], scoring=case["scoring"], bias=state["bias"],
                                      n_groups=case["groups"], top_groups=case["top_groups"],
                                      renormalize=case["renormalize"], scale=case["scale"])
        if not train:
            return [experts, weights]
        return [experts, weights.detach(), *torch.autograd.grad(weights, logits, state["grad"])]
    data = state["data"].detach().requires_grad_(train)
    if case["op"] == "dispatch":
        plan = povs.plan_rows(state["experts"], case["experts"])
        rows = povs.dispatch_rows(data, plan)
        out = [rows.detach(), plan.slots, plan.sources, plan.offsets]
        return out + [*torch.autograd.grad(rows, data, state["grad"])] if train else out
    weights = state["weights"].detach().requires_grad_(train)
    rows = povs.combine_rows(data, povs.RowPlan(*state["plan"]), weights)
    return [rows.detach(), *torch.autograd.grad(rows, (data, weights), state["grad"])] if train else [rows]


def run(state):
    if own:
        return _own_run(state)
    return {"sample": _sample, "route": _route, "dispatch": _dispatch, "combine": _combine}[state["case"]["op"]](state)


def work(case):
    rows = case["rows"]
    size = 4 if case["dtype"] == "float32" else 2
    if case["op"] == "sample":  # the scores once; subtract, scale, exponentiate, add
        return {"bytes": rows * case["width"] * size + 12 * rows, "flops": 4 * rows * case["width"]}
    if case["op"] == "route":
        n, k = case["experts"], case["k"]
        both = 2 if case["train"] else 1  # a training pass also writes the scores' gradient
        return {"bytes": rows * (both * n * size + k * (8 + 4 * (both - 1))), "flops": both * 6 * rows * n}
    k = min(case["k"], case["experts"])
    one, many = rows * case["width"], rows * k * case["width"]
    if case["op"] == "dispatch":  # rows read once, written k times; the gradient the other way round
        both = 2 if case["train"] else 1
        return {"bytes": both * (one + many) * size + 12 * rows * k, "flops": many if case["train"] else 0}
    if case["train"]:  # expert rows read once for both passes, their gradient written; rows out, their gradient in
        return {"bytes": (2 * one + 2 * many) * size + 16 * rows * k, "flops": 5 * many}
    return {"bytes": (one + many) * size + 8 * rows * k, "flops": 2 * many}


# ------------------------------------------------------------------------------------------
# The definitions in 64 bits, row by row or slot by slot.
# ------------------------------------------------------------------------------------------


def _exact_sample(state):
    case = state["case"]

    def of(name, r):
        value = state[name]
        return value[r].item() if isinstance(value, torch.Tensor) else value

    ids = []
    for r in range(case["rows"]):
        x = state["logits"][r].double()
        top, t = x.max(), of("temperature", r)
        if t <= 0:
            ids.append((x == top).nonzero()[0, 0])
            continue
        p = torch.exp((x - top) / t)
        # Candidates in order of their weight, then cut from behind by each rule.
        order = (-x).argsort(stable=True)
        k = of("top_k", r)
        order = order[:k] if k > 0 else order
        q = p[order] / p[order].sum()
        count = order.numel()
        if of("top_p", r) < 1:
            before = torch.cat([q.new_zeros(1), q.cumsum(0)[:-1]])
            count = max(1, int((before < of("top_p", r)).sum()))
        order = order[:count]
        order = order[p[order] >= of("min_p", r)]
        kept = order.sort().values
        running = p[kept].cumsum(0)
        at = torch.searchsorted(running, running[-1:] * state["uniforms"][r].double(), right=True)
        ids.append(kept[at.clamp(max=kept.numel() - 1)][0])
    return torch.stack([i.reshape(()) for i in ids]).to(torch.int64)


def _exact_route(state):
    import numpy as np

    case = state["case"]
    x = state["logits"].double().cpu().numpy()
    rows, n = x.shape
    if case["scoring"] == "softmax":
        s = np.exp(x - np.max(x, axis=1, keepdims=True))
        s /= np.sum(s, axis=1, keepdims=True)
    else:
        s = 1.0 / (1.0 + np.exp(-x))
    c = s.copy() if state["bias"] is None else s + state["bias"].double().cpu().numpy()
    if case["groups"] > 1:
        parts = c.reshape(rows, case["groups"], -1)
        ranked = np.sort(parts, axis=2)
        best = np.argsort(-(ranked[:, :, -1] + ranked[:, :, -2]), axis=1, kind="stable")[:, case["top_groups"]:]
        np.put_along_axis(parts, best[:, :, None], -np.inf, axis=1)
    e = np.argsort(-c, axis=1, kind="stable")[:, :case["k"]]
    w = np.take_along_axis(s, e, axis=1)
    total = w.sum(1, keepdims=True) if case["renormalize"] else 1.0
    out = [torch.from_numpy(e.astype(np.int32)), torch.from_numpy(w / total * case["scale"])]
    if case["train"]:
        # The Jacobian's product: dL/dx_i = sum over chosen j of dL/dw_j dw_j/dx_i.
        up = state["grad"].double().cpu().numpy() * case["scale"]
        hit = np.zeros((rows, n))
        np.put_along_axis(hit, e, up, axis=1)
        chosen = np.zeros((rows, n))
        np.put_along_axis(chosen, e, 1.0, axis=1)
        f = s * chosen / total  # the weights before scaling, zero elsewhere
        mean = (up * w / total).sum(1, keepdims=True)
        if case["scoring"] == "softmax":
            d = f * (hit - mean) if case["renormalize"] else f * hit - s * mean
        else:
            d = f * (1.0 - s) * (hit - (mean if case["renormalize"] else 0.0))
        out.append(torch.from_numpy(d))
    return out


def _exact_plan(experts, n_experts):
    import numpy as np

    e = experts.cpu().numpy().reshape(-1)
    slots = np.full(e.size, -1, dtype=np.int32)
    sources = np.full(e.size, -1, dtype=np.int32)
    offsets = np.zeros(n_experts + 1, dtype=np.int32)
    for x in range(n_experts):
        mine = np.flatnonzero(e == x)
        at = offsets[x] + np.arange(mine.size)
        slots[mine], sources[at] = at, mine
        offsets[x + 1] = offsets[x] + mine.size
    return (torch.from_numpy(slots.reshape(tuple(experts.shape))), torch.from_numpy(sources),
            torch.from_numpy(offsets))


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "sample":
        return _exact_sample(state)
    if case["op"] == "route":
        return _exact_route(state)
    plan = _exact_plan(state["experts"], case["experts"])
    slots = plan[0].cuda().long()
    data = state["data"].double()
    there = (slots >= 0).unsqueeze(2)
    if case["op"] == "dispatch":
        rows = data.new_zeros(slots.numel(), case["width"])
        for j in range(slots.shape[1]):
            rows[slots[:, j][there[:, j, 0]]] = data[there[:, j, 0]]
        out = [rows, *plan]
        if case["train"]:
            grad, total = state["grad"].double(), torch.zeros_like(data)
            for j in range(slots.shape[1]):
                total += torch.where(there[:, j], grad[slots[:, j].clamp(min=0)], 0.0)
            out.append(total)
        return out
    weights = state["weights"].double()
    total = data.new_zeros(case["rows"], case["width"])
    for j in range(slots.shape[1]):
        total += torch.where(there[:, j], data[slots[:, j].clamp(min=0)], 0.0) * weights[:, j:j + 1]
    out = [total]
    if case["train"]:
        grad = state["grad"].double()
        rows, dots = torch.zeros_like(data), torch.zeros_like(weights)
        for j in range(slots.shape[1]):
            m = there[:, j, 0]
            rows[slots[m, j]] = grad[m] * weights[m, j:j + 1]
            dots[m, j] = (grad[m] * data[slots[m, j]]).sum(1)
        out += [rows, dots]
    return out
