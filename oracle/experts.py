"""Routed experts in 64 bits (numpy) -- TEST INFRASTRUCTURE ONLY.

Restates what include/nsx.h says of nsx_expert_*: choice, plan, products, join, and their gradients, row by row and expert by
expert, without any code of the product."""
import numpy as np


def scores(x, sigmoid):
    """[T, E] float64 scores; -inf logits score 0; a row without a live expert is all 0."""
    x = np.asarray(x, np.float64)
    live = x > -np.inf
    if sigmoid:
        with np.errstate(over="ignore"):
            return np.where(live, 1.0 / (1.0 + np.exp(-x)), 0.0)
    m = np.where(live, x, -np.inf).max(axis=1, keepdims=True)
    e = np.where(live, np.exp(x - np.where(np.isfinite(m), m, 0.0)), 0.0)
    z = e.sum(axis=1, keepdims=True)
    return e / np.where(z > 0, z, 1.0)


def route(x, k, sigmoid=False, bias=None, n_groups=1, top_groups=None, group_top=1, renormalise=True, scale=1.0, selector=None):
    """(weights [T, k] float64, chosen [T, k] int32)."""
    x = np.asarray(x, np.float64)
    T, E = x.shape
    top_groups = n_groups if top_groups is None else top_groups
    weights, chosen = np.zeros((T, k)), np.full((T, k), -1, np.int32)
    for t in range(T):
        if selector is not None and not selector[t]:
            continue
        if np.isnan(x[t]).any() or (not sigmoid and np.isposinf(x[t]).any()):
            weights[t], chosen[t] = np.nan, np.arange(k)
            continue
        s = scores(x[t:t + 1], sigmoid)[0]
        c = s + (0.0 if bias is None else np.asarray(bias, np.float64))
        c = np.where(x[t] > -np.inf, c, -np.inf)
        if top_groups < n_groups:
            by = np.sort(c.reshape(n_groups, -1), axis=1)[:, ::-1][:, :group_top].sum(axis=1)
            on = np.zeros(n_groups, bool)
            on[np.argsort(-by, kind="stable")[:top_groups]] = True
            c = np.where(np.repeat(on, E // n_groups), c, -np.inf)
        order = [e for e in np.argsort(-c, kind="stable") if c[e] > -np.inf][:k]
        if not order:
            continue
        chosen[t, :len(order)] = order
        w = s[order]
        if renormalise:
            # ratios of the scores; where all of them underflow even 64 bits they are those of exp(x)
            if w.sum() == 0 or (w < 1e-290).all():
                w = np.exp(x[t, order] - x[t, order].max())
            w = w / w.sum()
        weights[t, :len(order)] = scale * w
    return weights, chosen


def route_bwd(x, weights, chosen, g, sigmoid=False, renormalise=True, scale=1.0):
    """Gradient of the logits, by the chain rule through the scores."""
    x = np.asarray(x, np.float64)
    d = np.zeros_like(x)
    s = scores(x, sigmoid)
    for t in range(x.shape[0]):
        on = [j for j in range(chosen.shape[1]) if chosen[t, j] >= 0]
        if not on:
            continue
        e, gt, w = chosen[t, on], g[t, on].astype(np.float64), weights[t, on]
        # dL / d log s of the chosen, then the score's own derivative
        dlog = w * (gt - (gt * w).sum() / scale) if renormalise else w * gt
        if sigmoid:
            d[t, e] = dlog * (1.0 - s[t, e])
        else:
            np.add.at(d[t], e, dlog)
            if not renormalise:
                d[t] -= s[t] * dlog.sum()
    return d


def plan(chosen, n_experts, n_rows=None):
    """(offsets, rows, positions) int32; rows behind ``n_rows`` are not routed."""
    T, k = chosen.shape
    flat = chosen.reshape(-1).copy()
    if n_rows is not None:
        flat[max(0, n_rows) * k:] = -1
    offsets, rows = np.zeros(n_experts + 1, np.int32), np.full(T * k, -1, np.int32)
    positions = np.full(T * k, -1, np.int32)
    at = 0
    for e in range(n_experts):
        mine = np.nonzero(flat == e)[0]
        rows[at:at + len(mine)] = mine
        positions[mine] = np.arange(at, at + len(mine))
        at += len(mine)
        offsets[e + 1] = at
    return offsets, rows, positions.reshape(T, k)


def linear(x, w, offsets, rows, k, gather, relu):
    """(y [R, N], sum of the terms' magnitudes [R, N]) float64."""
    x, w = np.asarray(x, np.float64), np.asarray(w, np.float64)
    y = np.zeros((len(rows), w.shape[1]))
    mag = np.zeros_like(y)
    for e in range(w.shape[0]):
        a, b = offsets[e], offsets[e + 1]
        src = x[rows[a:b] // k] if gather else x[a:b]
        y[a:b] = src @ w[e].T
        mag[a:b] = np.abs(src) @ np.abs(w[e]).T
    return (np.maximum(y, 0) if relu else y), mag


def linear_bwd(x, w, offsets, rows, k, gather, dz):
    """(dx in the plan's order, its magnitudes, dW, its magnitudes) of dz (dy where the ReLU let it through)."""
    x, w, dz = np.asarray(x, np.float64), np.asarray(w, np.float64), np.asarray(dz, np.float64)
    dx, mx = np.zeros((len(rows), w.shape[2])), np.zeros((len(rows), w.shape[2]))
    dw, mw = np.zeros_like(w), np.zeros_like(w)
    for e in range(w.shape[0]):
        a, b = offsets[e], offsets[e + 1]
        src = x[rows[a:b] // k] if gather else x[a:b]
        dx[a:b], mx[a:b] = dz[a:b] @ w[e], np.abs(dz[a:b]) @ np.abs(w[e])
        dw[e], mw[e] = dz[a:b].T @ src, np.abs(dz[a:b]).T @ np.abs(src)
    return dx, mx, dw, mw


def combine(y, weights, positions):
    """(out [T, N], magnitudes)."""
    y, weights = np.asarray(y, np.float64), np.asarray(weights, np.float64)
    out, mag = np.zeros((positions.shape[0], y.shape[1])), np.zeros((positions.shape[0], y.shape[1]))
    for j in range(positions.shape[1]):
        on = positions[:, j] >= 0
        term = weights[on, j, None] * y[positions[on, j]]
        out[on] += term
        mag[on] += np.abs(term)
    return out, mag
