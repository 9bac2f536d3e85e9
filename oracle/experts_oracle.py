"""NumPy float64 restatement of the mixture and distillation operators (test infrastructure): row by row, from the definitions."""
from __future__ import annotations

import numpy as np


def route(x, k, score="softmax", bias=None, n_groups=1, top_groups=None, group_score="max", renormalise=True, scale=1.0, mask=None):
    x = np.asarray(x, dtype=np.float64)
    n, e = x.shape
    top_groups = n_groups if top_groups is None else top_groups
    mask = np.ones((n, e), bool) if mask is None else np.broadcast_to(np.asarray(mask, bool), (n, e))
    experts, weights = np.full((n, k), -1, np.int32), np.zeros((n, k))
    for i in range(n):
        open_ = [c for c in range(e) if mask[i, c] and x[i, c] != -np.inf]
        if any(not x[i, c] < np.inf for c in open_):
            weights[i] = np.nan
            continue
        if bias is not None and any(not bias[c] < np.inf for c in open_):
            weights[i] = np.nan
            continue
        p = probabilities(x[i], open_, score)
        key = {c: p[c] + float(bias[c]) if bias is not None else x[i, c] for c in open_ if bias is None or bias[c] != -np.inf}
        if n_groups > 1:
            size = e // n_groups
            gs = []
            rank = key if bias is not None or group_score == "max" else {c: p[c] for c in open_}       # sums are sums of probabilities
            for g in range(n_groups):
                mine = sorted((rank[c] for c in key if c // size == g), reverse=True)
                gs.append(-np.inf if not mine else sum(mine[:2]) if group_score == "top2" else mine[0])
            keep = set(sorted(range(n_groups), key=lambda g: (-gs[g], g))[:top_groups])
            key = {c: v for c, v in key.items() if c // size in keep}
        chosen = sorted(key, key=lambda c: (-key[c], c))[:k]
        experts[i, :len(chosen)] = chosen
        if chosen:
            weights[i, :len(chosen)] = scale * chosen_weights(x[i], p, chosen, score, renormalise)
    return experts, weights


def log_sigmoid(t):
    return -np.logaddexp(0.0, -np.asarray(t, dtype=np.float64))


def probabilities(row, open_, score):
    p = np.zeros(len(row))
    if open_:
        if score == "sigmoid":
            p[open_] = np.exp(log_sigmoid(row[open_]))
        else:
            t = np.exp(row[open_] - row[open_].max())
            p[open_] = t / t.sum()
    return p


def chosen_weights(row, p, chosen, score, renormalise):
    if not renormalise:
        return p[chosen]
    t = log_sigmoid(row[chosen]) if score == "sigmoid" else row[chosen]
    t = np.exp(t - t.max())
    return t / t.sum()


def route_grad(x, experts, dweights, score="softmax", renormalise=True, scale=1.0, mask=None):
    """Chain rule written out with dense Jacobians."""
    x = np.asarray(x, dtype=np.float64)
    n, e = x.shape
    mask = np.ones((n, e), bool) if mask is None else np.broadcast_to(np.asarray(mask, bool), (n, e))
    dx = np.zeros((n, e))
    for i in range(n):
        open_ = [c for c in range(e) if mask[i, c] and x[i, c] != -np.inf]
        js = [j for j in range(experts.shape[1]) if 0 <= experts[i, j] < e]
        if not js:
            continue
        chosen = [int(experts[i, j]) for j in js]
        g = scale * np.asarray([dweights[i, j] for j in js], dtype=np.float64)
        p = probabilities(x[i], open_, score)
        if renormalise:
            r = chosen_weights(x[i], p, chosen, score, True)
            dt = r * (g - (r * g).sum())                                 # with respect to log p of the chosen, up to a constant
            dx[i, chosen] += dt * (np.exp(log_sigmoid(-x[i, chosen])) if score == "sigmoid" else 1.0)
        elif score == "sigmoid":
            dx[i, chosen] += g * p[chosen] * np.exp(log_sigmoid(-x[i, chosen]))
        else:
            dp = np.zeros(e)
            dp[chosen] = g
            dx[i] = p * (dp - (p * dp).sum())
    return dx


def plan(experts, n_experts):
    ex = np.asarray(experts)
    flat = ex.reshape(-1)
    k = ex.shape[1] if ex.ndim == 2 else 1
    places = [(int(c), s) for s, c in enumerate(flat) if 0 <= c < n_experts]
    places.sort()                                                        # by expert, then by slot
    rows, positions = np.full(flat.size, -1, np.int32), np.full(flat.size, -1, np.int32)
    for at, (_, s) in enumerate(places):
        rows[at], positions[s] = s // k, at
    counts = np.bincount([c for c, _ in places], minlength=n_experts).astype(np.int32)
    offsets = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
    return rows, positions.reshape(ex.shape), counts, offsets


def dispatch(X, rows):
    X = np.asarray(X, dtype=np.float64)
    return np.where((rows >= 0)[:, None], X[np.maximum(rows, 0)], 0.0)


def combine(F, weights, positions):
    F = np.asarray(F, dtype=np.float64)
    n, k = positions.shape
    y = np.zeros((n, F.shape[1]))
    for i in range(n):
        for j in range(k):
            with np.errstate(invalid="ignore"):              # no place: the weight times a row of zeros
                y[i] += weights[i, j] * (F[positions[i, j]] if positions[i, j] >= 0 else 0.0)
    return y


def combine_grad(F, weights, positions, dout):
    F, dout = np.asarray(F, dtype=np.float64), np.asarray(dout, dtype=np.float64)
    dF, dw = np.zeros_like(F), np.zeros(positions.shape)
    for (i, j), at in np.ndenumerate(positions):
        if at >= 0:
            dF[at] = weights[i, j] * dout[i]
            dw[i, j] = dout[i] @ F[at]
    return dF, dw


def _logsumexp(t):
    t = np.asarray(t, dtype=np.float64)
    if t.size == 0:
        return -np.inf
    m = t.max()
    return m if m == -np.inf else m + np.log(np.exp(t - m).sum())


def distill(logits, top, index, top_lse=None, temperature=1.0, direction="forward", row_weight=None, resolution=2.0 ** -53):
    """(loss, gradient, scale): scale[n] bounds the sum of the magnitudes of the divergence's terms, for tolerances."""
    x = np.asarray(logits, dtype=np.float64)
    n, v = x.shape
    loss, grad, size = np.zeros(n), np.zeros((n, v)), np.zeros(n)
    for i in range(n):
        w = 1.0 if row_weight is None else float(row_weight[i])
        if w == 0.0:
            continue
        entries = [(int(c), float(t)) for c, t in zip(index[i], top[i]) if c != -1 and t != -np.inf]
        if any(not 0 <= c < v for c in index[i] if c != -1):
            loss[i], grad[i] = np.nan, np.nan
            continue
        if not entries:
            continue
        classes = sorted({c for c, _ in entries})
        lp = np.array([_logsumexp([t / temperature for c2, t in entries if c2 == c]) for c in classes])
        lp = lp - (_logsumexp(lp) if top_lse is None else float(top_lse[i]))
        lq = (x[i] - x[i].max()) / temperature               # from the maximum: log V is lost next to the types' lowest values
        lq = lq - _logsumexp(lq)
        outside = np.ones(v, bool)
        outside[classes] = False
        p, lqt = np.exp(lp), lq[classes]
        rest = top_lse is not None and outside.any()
        pr = max(0.0, 1.0 - p.sum()) if rest else 0.0
        lqr = _logsumexp(lq[outside]) if rest else 0.0
        factor = temperature ** 2 * w
        with np.errstate(divide="ignore", invalid="ignore"):
            if direction == "forward":
                terms = np.where(p > 0, p * (lp - lqt), 0.0)
                kl = terms.sum() + (pr * (np.log(pr) - lqr) if pr > 0 else 0.0)
                ratio = np.exp(np.log(pr) - lqr) if pr > 0 else 0.0
                total = p.sum() + pr                             # the teacher's mass; 1 within what single precision leaves of top_lse
                total = 1.0 if abs(total - 1.0) < 2.0 ** -18 else total
                grad[i] = np.exp(lq) * (total - ratio)
                grad[i, classes] = np.exp(lqt) * total - p
                size[i] = factor * (np.abs(p * lp).sum() + np.abs(p * lqt).sum() + abs(pr * lqr) + 1.0 + ratio)
            else:
                q, qr = np.exp(lqt), np.exp(lqr) if rest else 0.0
                lr = lqr - np.log(max(pr, resolution)) if rest else 0.0
                terms = np.where(q != 0, q * (lqt - lp), 0.0)
                kl = terms.sum() + (qr * lr if qr != 0 else 0.0)
                grad[i] = np.exp(lq) * (lr - kl)
                grad[i, classes] = np.where(q != 0, q * (lqt - lp - kl), 0.0)
                size[i] = factor * (np.abs(q * lqt).sum() + np.abs(q * lp).sum() + qr * (abs(lr) + abs(lqr)) + 1.0)
        if not np.isfinite(size[i]):                         # an infinite divergence: the terms that are finite
            size[i] = factor * (1.0 + np.nan_to_num(np.abs(p * lp), posinf=0.0).sum() + (ratio if direction == "forward" else 0.0))
        loss[i] = factor * kl
        grad[i] *= temperature * w
    return loss, grad, size
