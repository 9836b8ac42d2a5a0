"""Plain double-precision routing (test infrastructure): one token at a time, straight from the
definition in include/hymoe.h, for the tests of hymoe_route and hymoe_route_backward."""
from __future__ import annotations

import numpy as np

BIG = float(np.finfo(np.float32).max)


def clean(v) -> np.ndarray:
    """Logits (or biases) as the definition takes them: NaN closes, +inf is FLT_MAX."""
    v = np.asarray(v, np.float64)
    return np.minimum(np.where(np.isnan(v), -np.inf, v), BIG)


def log_scores(z, score: str) -> np.ndarray:
    """Logarithm of every score of one token; -inf for closed experts."""
    open_ = z > -np.inf
    out = np.full(z.shape, -np.inf)
    if not open_.any():
        return out
    if score == "sigmoid":
        out[open_] = -np.logaddexp(0.0, -z[open_])
    else:
        m = z[open_].max()
        out[open_] = z[open_] - m - np.log(np.exp(z[open_] - m).sum())
    return out


def route_row(z, bias, K, score, group, group_score, norm, scale):
    """(idx [K], weights [K], scores [E]) of one token's clean logits."""
    E = len(z)
    ls = log_scores(z, score)
    s = np.exp(ls)
    open_ = z > -np.inf
    b = None if bias is None else clean(bias)
    c = np.where(open_, z if b is None else s + b, -np.inf)
    if group:
        ng, tg = group
        base = np.where(open_, s, -np.inf) if b is None and group_score == "top2" else c
        val = []
        for g in range(ng):
            v = np.sort(base[g * (E // ng):(g + 1) * (E // ng)])[::-1]
            v = v[v > -np.inf]
            val.append(-np.inf if len(v) == 0 else v[0] if group_score == "max" or len(v) == 1 else v[0] + v[1])
        kept = sorted(range(ng), key=lambda g: (-val[g], g))[:tg]
        for g in range(ng):
            if g not in kept:
                c[g * (E // ng):(g + 1) * (E // ng)] = -np.inf
    order = [e for e in sorted(range(E), key=lambda e: (-c[e], e)) if c[e] > -np.inf][:K]
    idx = np.full(K, -1, np.int64)
    w = np.zeros(K)
    idx[:len(order)] = order
    if order:
        lw = ls[order]
        if norm:
            if score == "softmax":  # the common sum drops out
                lw = z[order]
            lw = lw - lw.max()
            w[:len(order)] = np.exp(lw) / np.exp(lw).sum()
        else:
            w[:len(order)] = s[order]
    return idx, w * scale, s


def route(z, bias, K, score="softmax", group=None, group_score="max", norm=True, scale=1.0):
    rows = [route_row(r, bias, K, score, group, group_score, norm, scale) for r in clean(z)]
    E = np.asarray(z).shape[1]
    idx = np.array([r[0] for r in rows], np.int64).reshape(-1, K)
    return {"idx": idx, "weights": np.array([r[1] for r in rows]).reshape(-1, K),
            "scores": np.array([r[2] for r in rows]).reshape(-1, E),
            "counts": np.bincount(idx[idx >= 0], minlength=E)}


def weights_of(z, idx, score, norm, scale):
    """Weights [K] of given selections of one token (entries that take no part: 0) and its scores."""
    E = len(z)
    s = np.exp(log_scores(z, score))
    ok = np.array([0 <= e < E and z[max(0, min(E - 1, e))] > -np.inf for e in idx])
    sel = np.where(ok, s[np.clip(idx, 0, E - 1)], 0.0)
    if norm:
        t = sel.sum()
        sel = sel / t if t > 0 else sel
    return sel * scale, s


def loss(z, idx, dw, ds, score, norm, scale):
    w, s = weights_of(z, idx, score, norm, scale)
    return float((w * dw).sum() + (0.0 if ds is None else (s * np.where(z > -np.inf, ds, 0.0)).sum()))


def grad_row(z, idx, dw, ds, score, norm, scale):
    """Formula of the gradient of `loss` to the logits, and the sum of its terms' magnitudes."""
    E = len(z)
    z = clean(z)
    s = np.exp(log_scores(z, score))
    open_ = z > -np.inf
    ok = np.array([0 <= e < E and z[max(0, min(E - 1, e))] > -np.inf for e in idx])
    sel = np.where(ok, s[np.clip(idx, 0, E - 1)], 0.0)
    g = np.where(ok, dw * scale, 0.0)
    size = np.abs(g) * sel
    if norm:
        n = sel / sel.sum() if sel.sum() > 0 else sel
        term = n * (g - (g * n).sum())
        size = n * (np.abs(g) + (np.abs(g) * n).sum())
    else:
        term = g * sel
    dss = np.zeros(E) if ds is None else np.where(open_, ds, 0.0)
    t = dss * s
    mag = np.abs(t)
    np.add.at(t, np.clip(idx, 0, E - 1)[ok], term[ok])
    np.add.at(mag, np.clip(idx, 0, E - 1)[ok], size[ok])
    if score == "sigmoid":
        d = t * np.exp(-np.logaddexp(0.0, z))
    else:
        d = t - s * t.sum()
        mag = mag + s * mag.sum()
    return np.where(open_, d, 0.0), mag
