"""The row operators (``povs.sample``, ``route``, ``plan_rows``, ``dispatch_rows``, ``combine_rows``) from their
definitions, in NumPy and 64 bits, one row at a time."""

from __future__ import annotations

import numpy as np


def sample_row(x: np.ndarray, u: float, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0) -> int:
    x = np.where(np.isnan(x), -np.inf, x.astype(np.float64))
    if not (x > -np.inf).any():
        return -1
    order = np.argsort(-x, kind="stable")
    order = order[x[order] > -np.inf]
    if not temperature > 0:
        return int(order[0])
    top = x[order[0]]
    w = np.ones_like(x) * (x == top) if np.isinf(top) else np.exp((x - top) / temperature)
    if 0 < top_k < len(order):
        order = order[:top_k]
    if top_p < 1:
        running = np.concatenate([[0.0], np.cumsum(w[order])])
        keep = running[:-1] < top_p * running[-1]
        keep[0] = True
        order = order[keep]
    keep = (w[order] >= min_p) | (x[order] == top)
    kept = np.sort(order[keep])
    running = np.cumsum(w[kept])
    target = min(max(u, 0.0), 1.0) * running[-1]
    above = np.flatnonzero(running > target)
    last = np.flatnonzero(w[kept] > 0)[-1]
    return int(kept[above[0] if len(above) else last])


def _rank(values: np.ndarray) -> np.ndarray:
    """Places by descending value, equal ones by the lowest place, NaN behind every number."""
    nan = np.isnan(values)
    return np.lexsort((np.arange(len(values)), -np.where(nan, 0.0, values), nan))


def scores(x: np.ndarray, scoring: str) -> np.ndarray:
    x = x.astype(np.float64)
    with np.errstate(all="ignore"):
        if scoring == "sigmoid":
            return 1 / (1 + np.exp(-x))
        top = np.max(x[~np.isnan(x)], initial=-np.inf)
        if top == -np.inf:
            return np.where(np.isnan(x), np.nan, 0.0) if not np.isnan(x).any() else np.where(x == -np.inf, 0.0, np.nan)
        e = np.exp(x - top)
        return np.where(x == -np.inf, 0.0, e / e.sum())


def route_row(x, top_k, scoring="softmax", bias=None, n_groups=1, top_groups=None, group_score="top2",
              renormalize=False, scale=1.0):
    n = len(x)
    s = scores(x, scoring)
    with np.errstate(all="ignore"):
        c = s if bias is None else s + bias.astype(np.float64)
        if bias is None and (top_groups is None or top_groups == n_groups):
            c = np.where(np.isnan(s), np.nan, x)  # scores rise with the logits
        c = np.where(x == -np.inf, -np.inf, c)
        if top_groups is not None and top_groups < n_groups:
            parts = c.reshape(n_groups, -1)
            best = [p[_rank(p)[: 2 if group_score == "top2" else 1]].sum() for p in parts]
            kept = np.zeros(n_groups, dtype=bool)
            kept[_rank(np.array(best))[:top_groups]] = True
            c = np.where(np.repeat(kept, n // n_groups), c, -np.inf)
        order = [e for e in _rank(np.where(c == -np.inf, np.nan, c)) if c[e] != -np.inf]
        # NaN scores rank behind the numbers and before what cannot be chosen.
        order = [e for e in order if not np.isnan(c[e])] + [e for e in order if np.isnan(c[e])]
        chosen = order[:top_k]
        w = s[chosen] * scale
        if renormalize:
            total = s[chosen].sum()
            w = np.zeros_like(w) if total == 0 else w / total
    missing = top_k - len(chosen)
    return np.array(chosen + [-1] * missing, dtype=np.int32), np.concatenate([w, np.zeros(missing)])


def route(x, top_k, **kw):
    rows = [route_row(r, top_k, **kw) for r in x]
    return np.stack([e for e, _ in rows]), np.stack([w for _, w in rows])


def weights_of(x, experts, scoring, renormalize, scale):
    """The weights as a function of the logits for fixed choices (rows without -1)."""
    s = np.stack([scores(r, scoring) for r in x])
    w = np.take_along_axis(s, experts, 1) * scale
    return w / (w.sum(1, keepdims=True) / scale) if renormalize else w


def route_gradient(x, experts, g, scoring, renormalize, scale):
    """(gradient of the logits, a bound on the size of the terms that make each of its numbers)."""
    s = np.stack([scores(r, scoring) for r in x])
    out, size = np.zeros_like(s), np.zeros_like(s)
    for r in range(len(x)):
        here = experts[r] >= 0
        e = experts[r][here]
        f, up = s[r, e], g[r][here].astype(np.float64) * scale
        total = f.sum() if renormalize else 1.0
        df, mag = up / total, np.abs(up) / total
        if renormalize:
            df = df - (up * f).sum() / total**2
            mag = mag + (np.abs(up) * f).sum() / total**2
        full, fmag = np.zeros(s.shape[1]), np.zeros(s.shape[1])
        full[e], fmag[e] = df, mag
        if scoring == "softmax":
            out[r] = s[r] * (full - (f * df).sum())
            size[r] = s[r] * (fmag + (f * mag).sum())
        else:
            out[r] = s[r] * (1 - s[r]) * full
            size[r] = s[r] * fmag
    return out, size


def plan(experts: np.ndarray, n_experts: int):
    flat = experts.reshape(-1)
    slots, sources = np.full(flat.size, -1, np.int32), np.full(flat.size, -1, np.int32)
    offsets, at = [0], 0
    for e in range(n_experts):
        for i in np.flatnonzero(flat == e):
            slots[i], sources[at] = at, i
            at += 1
        offsets.append(at)
    return slots.reshape(experts.shape), sources, np.array(offsets, np.int32)


def dispatch(data: np.ndarray, slots: np.ndarray) -> np.ndarray:
    out = np.zeros((slots.size, *data.shape[1:]), data.dtype)
    for r, j in zip(*np.nonzero(slots >= 0)):
        out[slots[r, j]] = data[r]
    return out


def combine(data: np.ndarray, slots: np.ndarray, weights: np.ndarray | None):
    """(sums, sums of the absolute values), in 64 bits."""
    out = np.zeros((slots.shape[0], *data.shape[1:]))
    size = np.zeros_like(out)
    for r, j in zip(*np.nonzero(slots >= 0)):
        term = data[slots[r, j]].astype(np.float64) * (1.0 if weights is None else float(weights[r, j]))
        out[r] += term
        size[r] += np.abs(term)
    return out, size
