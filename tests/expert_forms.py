"""Root-mean-square norm, routing and experts' products in 64 bits, from their
definitions (numpy on the CPU), for the tests of ien_rms_norm, ien_route and
ien_experts_in8 / _out8."""

import numpy as np

import eight_bits as E


def rms_norm(s, gamma, eps):
    """f64 norm of the rows s."""
    s = s.astype(np.float64)
    y = s / np.sqrt((s * s).mean(1, keepdims=True) + eps)
    return y if gamma is None else y * gamma.astype(np.float64)


def scores(logits, softmax):
    """f64 scores; NaN and -inf count as no expert's (0)."""
    v = logits.astype(np.float64)
    v = np.where(np.isnan(v), -np.inf, v)
    if not softmax:
        return np.where(v > 0, 1 / (1 + np.exp(-np.abs(v))), np.exp(-np.abs(v)) / (1 + np.exp(-np.abs(v))))
    m = v.max(1, keepdims=True)
    m = np.where(m > -np.inf, m, 0)
    with np.errstate(invalid="ignore"):
        e = np.where(v == m, 1.0, np.exp(v - m))
    total = e.sum(1, keepdims=True)
    return np.divide(e, total, out=np.zeros_like(e), where=total > 0)


def route(logits, top, softmax=True, bias=None, groups=1, kept=None, group_top=1, renormalise=True, scale=1.0):
    """(index [t, top], weight f64): one token and one choice at a time."""
    kept = groups if kept is None else kept
    s = scores(logits, softmax)
    tokens, experts = s.shape
    per = experts // groups
    index, weight = np.full((tokens, top), -1), np.zeros((tokens, top))
    for t in range(tokens):
        choice = {}
        for e in range(experts):
            b = 0.0 if bias is None else float(bias[e])
            if logits[t, e] > -np.inf and b > -np.inf:  # (NaN: no)
                choice[e] = s[t, e] + b
        ranks = []
        for g in range(groups):
            best = sorted((choice[e] for e in range(g * per, (g + 1) * per) if e in choice), reverse=True)[:group_top]
            if best:
                ranks.append((-sum(best), g))
        open_ = {g for _, g in sorted(ranks)[:kept]}
        order = sorted((-c, e) for e, c in choice.items() if e // per in open_)[:top]
        for k, (_, e) in enumerate(order):
            index[t, k], weight[t, k] = e, s[t, e]
    if renormalise:
        total = weight.sum(1, keepdims=True)
        weight = np.divide(weight, total, out=np.zeros_like(weight), where=total > 0)
    return index, weight * scale


def plan(index, experts):
    """(offsets, order): pairs by expert, those without one last."""
    flat = index.reshape(-1)
    flat = np.where((flat < 0) | (flat >= experts), experts, flat)
    offsets = np.concatenate([[0], np.cumsum(np.bincount(flat, minlength=experts + 1)[:experts])])
    return offsets, np.argsort(flat, kind="stable")


def weights(w):
    """f64 values of weights [experts, c, n] in 8 bits."""
    return np.stack([E.weights(m, 1) for m in w])


def products(x, index, w, b, gather):
    """f64 rows [pairs, n] in the plan's order (pairs with an expert) and the magnitudes of their products' sums;
    x: rows a token (gather), or a pair in the plan's order."""
    tokens, top = index.shape
    offsets, order = plan(index, w.shape[0])
    y, size = np.zeros((offsets[-1], w.shape[2])), np.zeros((offsets[-1], w.shape[2]))
    for e in range(w.shape[0]):
        at = slice(offsets[e], offsets[e + 1])
        rows = x[order[at] // top] if gather else x[at]
        y[at] = rows @ w[e] + (0 if b is None else b[e])
        size[at] = np.abs(rows) @ np.abs(w[e]) + (0 if b is None else np.abs(b[e]))
    return y, size


def gate(v, act, gated):
    half = v.shape[1] // 2
    return E.activate(v[:, :half], act) * v[:, half:] if gated else E.activate(v, act)


def combine(y, index, weight, experts):
    """Each token's weighted sum of its pairs' rows (the plan's order)."""
    tokens, top = index.shape
    offsets, order = plan(index, experts)
    out = np.zeros((tokens, y.shape[1]))
    for p, pair in enumerate(order[:offsets[-1]]):
        out[pair // top] += np.float64(weight[pair // top, pair % top]) * y[p]
    return out
