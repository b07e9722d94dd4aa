"""Plain 64-bit statements of the operators past the cube (recurrence, router, experts' product), row by row, with bounds on what
rounding may do to them: test infrastructure, no code in common with the library."""
import math

import numpy as np

U64 = 2.0**-53


def sequences(offsets, n):
    return [(0, n)] if offsets is None else [(int(a), int(b)) for a, b in zip(offsets[:-1], offsets[1:])]


def gates(form, gate, d):
    g = np.repeat(np.asarray(gate, dtype=np.float64), d // gate.shape[1], axis=1)
    if form == "value":
        return g, np.ones_like(g)
    return np.exp(g), (np.sqrt(-np.expm1(2.0 * g)) if form == "stationary" else np.ones_like(g))


def recurrence(form, gate, x, offsets, h0):
    """-> (h, last, size of h's terms, longest sequence): rows of no sequence are NaN in h"""
    n, d = x.shape
    a, c = gates(form, gate, d)
    x = np.asarray(x, dtype=np.float64)
    seqs = sequences(offsets, n)
    h, size = np.full((n, d), np.nan), np.zeros((n, d))
    last, last_size = np.zeros((len(seqs), d)), np.zeros((len(seqs), d))
    for s, (lo, hi) in enumerate(seqs):
        v = np.zeros(d) if h0 is None else np.asarray(h0[s], dtype=np.float64)
        z = np.abs(v)
        for r in range(lo, hi):
            v = a[r] * v + c[r] * x[r]
            z = np.abs(a[r]) * z + np.abs(c[r] * x[r])
            h[r], size[r] = v, z
        last[s], last_size[s] = v, z
    return h, last, size, last_size


def recurrence_backward(form, gate, x, h, dh, offsets, h0, dlast):
    """-> dict of (value, size of its terms)"""
    n, d = dh.shape
    cols = gate.shape[1]
    a, c = gates(form, gate, d)
    f = lambda v: np.asarray(v, dtype=np.float64)  # noqa: E731
    h, dh = f(h), f(dh)
    x = f(x) if x is not None else np.zeros((n, d))
    seqs = sequences(offsets, n)
    dg, dgz, dx, dxz = (np.full((n, d), np.nan), np.zeros((n, d)), np.full((n, d), np.nan), np.zeros((n, d)))
    dh0, dh0z = np.zeros((len(seqs), d)), np.zeros((len(seqs), d))
    for s, (lo, hi) in enumerate(seqs):
        q = np.zeros(d) if dlast is None else f(dlast[s])
        z = np.abs(q)
        for r in range(hi - 1, lo - 1, -1):
            g, gz = dh[r] + q, np.abs(dh[r]) + z
            before = h[r - 1] if r > lo else (np.zeros(d) if h0 is None else f(h0[s]))
            dx[r], dxz[r] = c[r] * g, np.abs(c[r]) * gz
            v, vz = g * before, gz * np.abs(before)
            if form != "value":
                v, vz = v * a[r], vz * a[r]
            if form == "stationary":
                with np.errstate(divide="ignore", invalid="ignore"):
                    slope = np.where(c[r] > 0, a[r] * a[r] / c[r], 0.0)
                v, vz = v - g * x[r] * slope, vz + gz * np.abs(x[r]) * slope
            dg[r], dgz[r] = v, vz
            q, z = a[r] * g, np.abs(a[r]) * gz
        dh0[s], dh0z[s] = q, z
    shared = lambda m: m.reshape(n, cols, d // cols).sum(axis=2)  # noqa: E731
    return {"dgate": (shared(dg), shared(dgz)), "dx": (dx, dxz), "dh0": (dh0, dh0z)}


def scores(score, logits):
    z = np.asarray(logits, dtype=np.float64)
    if score == "sigmoid":
        with np.errstate(over="ignore"):
            return 1.0 / (1.0 + np.exp(-z))
    top = z.max(axis=1, keepdims=True)
    p = np.exp(z - np.where(np.isinf(top), 0.0, top))
    total = p.sum(axis=1, keepdims=True)
    return p / np.where(total == 0, 1.0, total)


def route(score, logits, bias, groups, top_groups, k, renormalise, scale):
    """-> (experts, weights, counts), one row at a time"""
    z = np.asarray(logits, dtype=np.float64)
    n, experts = z.shape
    p = scores(score, np.where(np.isnan(z), 0.0, z))
    chosen, weights = np.full((n, k), -1, dtype=np.int32), np.zeros((n, k))
    size = experts // groups
    for r in range(n):
        if np.isnan(z[r]).any() or (score == "softmax" and np.isposinf(z[r]).any()):
            weights[r] = np.nan
            continue
        rank = p[r] + bias if bias is not None else p[r]
        key = rank if bias is not None else z[r]
        open_ = np.ones(experts, dtype=bool) if bias is None else ~np.isnan(bias)
        open_ &= ~np.isneginf(z[r])
        if top_groups < groups:
            values = []
            for g in range(groups):
                mine = sorted((rank[e] for e in range(g * size, (g + 1) * size) if open_[e]), reverse=True)[:2]
                values.append(sum(mine) if mine else -math.inf)
            kept = sorted(range(groups), key=lambda g: (-values[g], g))[:top_groups]
            open_ &= np.array([e // size in kept for e in range(experts)])
        order = sorted((e for e in range(experts) if open_[e]), key=lambda e: (-key[e], e))[:k]
        chosen[r, :len(order)] = order
        w = p[r][order]
        if renormalise:
            w = w / w.sum() if w.sum() > 0 else 0.0 * w
        weights[r, :len(order)] = scale * w
    return chosen, weights, np.bincount(chosen[chosen >= 0].ravel(), minlength=experts)


def route_backward(score, logits, chosen, dweights, renormalise, scale):
    """-> (dlogits, size of its terms)"""
    z = np.asarray(logits, dtype=np.float64)
    n, experts = z.shape
    p = scores(score, z)
    out, size = np.zeros((n, experts)), np.zeros((n, experts))
    for r in range(n):
        used = [(j, e) for j, e in enumerate(chosen[r]) if 0 <= e < experts]
        total = sum(p[r, e] for _, e in used)
        ds, dz = np.zeros(experts), np.zeros(experts)
        mean = sum(p[r, e] / total * scale * dweights[r, j] for j, e in used) if renormalise and total > 0 else 0.0
        means = sum(abs(p[r, e] / total * scale * dweights[r, j]) for j, e in used) if renormalise and total > 0 else 0.0
        for j, e in used:
            w = scale * dweights[r, j]
            if renormalise:
                ds[e] += (w - mean) / total if total > 0 else 0.0
                dz[e] += (abs(w) + means) / total if total > 0 else 0.0
            else:
                ds[e] += w
                dz[e] += abs(w)
        if score == "sigmoid":
            out[r], size[r] = ds * p[r] * (1 - p[r]), dz * p[r] * (1 - p[r])
        else:
            out[r] = p[r] * (ds - (ds * p[r]).sum())
            size[r] = p[r] * (dz + (dz * p[r]).sum())
    return out, size


def covariance(spec, A, B):
    """k(a, b) for all pairs, from the differences"""
    name = spec[0]
    if name in ("sum", "prod"):
        a, b = covariance(spec[1], A, B), covariance(spec[2], A, B)
        return a + b if name == "sum" else a * b
    if name == "linear":
        return A @ B.T + spec[1]
    s = np.zeros((len(A), len(B)))
    for f in range(A.shape[1]):
        s += (A[:, None, f] - B[None, :, f]) ** 2
    if name == "squared_exp":
        return abs(spec[2]) * np.exp(-s / (2 * spec[1] ** 2))
    if name == "exponential":
        return abs(spec[2]) * np.exp(-np.sqrt(s) / (2 * spec[1] ** 2))
    t = np.sqrt(s) / abs(spec[1])
    if name == "matern1":
        return abs(spec[2]) * (1 + math.sqrt(3) * t) * np.exp(-math.sqrt(3) * t)
    if name == "matern2":
        return abs(spec[2]) * (1 + math.sqrt(5) * t + 5 * t * t / 3) * np.exp(-math.sqrt(5) * t)
    if name == "rational_quadratic":
        return (1 + s / (2 * spec[1] * spec[2] ** 2)) ** -spec[1]
    raise ValueError(name)


def experts_predict(spec, X, alpha, offsets, Xq, chosen, weights, prior):
    """-> (mean, slots, size of each slot's terms)"""
    m, k = chosen.shape
    slots, size = np.zeros((m, k)), np.zeros((m, k))
    for q in range(m):
        for j in range(k):
            e = chosen[q, j]
            if 0 <= e < len(offsets) - 1:
                lo, hi = offsets[e], offsets[e + 1]
                c = covariance(spec, Xq[q:q + 1], X[lo:hi])[0]
                slots[q, j], size[q, j] = c @ alpha[lo:hi], np.abs(c) @ np.abs(alpha[lo:hi])
    mean = (weights * slots).sum(axis=1) + (0.0 if prior is None else prior)
    return mean, slots, size


def experts_backward(spec, X, offsets, Xq, chosen, weights, slots, dmean):
    """-> (dweights, dalpha, size of dalpha's terms)"""
    m, k = chosen.shape
    E = len(offsets) - 1
    dw, da, size = np.zeros((m, k)), np.zeros(len(X)), np.zeros(len(X))
    for q in range(m):
        for j in range(k):
            e = chosen[q, j]
            if 0 <= e < E:
                lo, hi = offsets[e], offsets[e + 1]
                dw[q, j] = dmean[q] * slots[q, j]
                c = covariance(spec, Xq[q:q + 1], X[lo:hi])[0]
                da[lo:hi] += dmean[q] * weights[q, j] * c
                size[lo:hi] += np.abs(dmean[q] * weights[q, j] * c)
    return dw, da, size
