"""Routing to experts, sorting by expert, combining and low-rank adapters in 64 bits, from the definitions (include/eif_hip_moe.h,
include/eif_hip_adapters.h)."""
import numpy as np

MOST = np.float64(np.finfo(np.float32).max)
SOFTMAX, SIGMOID = 0, 1


def route(logits, top_k, score=SOFTMAX, bias=None, groups=1, groups_kept=1, group_best=1, renormalise=True, scale=1.0):
    """(ids [T, top_k] int32, weights [T, top_k] float64), a token at a time."""
    logits = np.asarray(logits, np.float64)
    tokens, experts = logits.shape
    ids, weights = np.full((tokens, top_k), -1, np.int32), np.zeros((tokens, top_k))
    with np.errstate(over="ignore"):
        for t in range(tokens):
            l = np.where(np.isnan(logits[t]), -np.inf, np.minimum(logits[t], MOST))
            has = l > -np.inf   # a score
            if not has.any():
                continue
            if score == SOFTMAX:
                s = np.where(has, np.exp(l - l[has].max()), 0.0)
                s = s / s.sum()
            else:
                s = 1.0 / (1.0 + np.exp(-l))
            b = np.zeros(experts) if bias is None else np.asarray(bias, np.float64)
            open_ = has & (b > -np.inf)
            v = np.where(open_, s + np.where(open_, b, 0.0), -np.inf)
            by = np.where(open_, l, -np.inf) if bias is None else v
            size = experts // groups
            if groups_kept < groups:
                worth = np.empty(groups)
                for g in range(groups):
                    part = slice(g * size, (g + 1) * size)
                    if group_best == 1:
                        worth[g] = by[part].max()
                    else:
                        two = np.sort(v[part])[::-1][:2]
                        worth[g] = two[0] if two[0] == -np.inf else two[two > -np.inf].sum()
                kept = sorted(range(groups), key=lambda g: (-worth[g], g))[:groups_kept]
                inside = np.isin(np.arange(experts) // size, kept)
                by = np.where(inside, by, -np.inf)
            order = [e for e in np.argsort(-by, kind="stable")[:top_k] if by[e] > -np.inf]
            n = len(order)
            if not n:
                continue
            ids[t, :n] = order
            if renormalise and score == SOFTMAX:
                w = np.exp(l[order] - l[order].max())
                w = w / w.sum()
            else:
                w = s[order]
                if renormalise:
                    w = w / w.sum() if w.sum() > 0 else np.zeros(n)
            weights[t, :n] = w * np.float64(np.float32(scale))
    return ids, weights


def sort(ids, experts, tail=-7):
    """offsets, row (with `tail` behind the last pair), slot."""
    flat = np.asarray(ids).reshape(-1)
    top = np.asarray(ids).shape[1]
    live = (flat >= 0) & (flat < experts)
    order = [p for p in np.argsort(np.where(live, flat, experts), kind="stable") if live[p]] if flat.size < 5000 else None
    if order is None:
        order = np.argsort(np.where(live, flat, experts), kind="stable")[:int(live.sum())]
    order = np.asarray(order, np.int64)
    offsets = np.concatenate([[0], np.cumsum(np.bincount(flat[live], minlength=experts))]).astype(np.int32)
    row, slot = np.full(flat.size, tail, np.int32), np.full(flat.size, -1, np.int32)
    row[:order.size] = order // top
    slot[order] = np.arange(order.size)
    return offsets, row, slot


def combine(y, slot, weights=None, add=None):
    """(out, sum of magnitudes) in float64; slot [T, K]."""
    y, (tokens, top) = np.asarray(y, np.float64), slot.shape
    out, mag = np.zeros((tokens, y.shape[1])), np.zeros((tokens, y.shape[1]))
    if add is not None:
        out += add
        mag += np.abs(add)
    for k in range(top):
        ok = (slot[:, k] >= 0) & (slot[:, k] < y.shape[0])
        part = y[slot[ok, k]] * (1.0 if weights is None else np.asarray(weights, np.float64)[ok, k, None])
        out[ok] += part
        mag[ok] += np.abs(part)
    return out, mag


def adapters(x, slot, pairs, base, rows):
    """(y, tolerance) for pairs {slot: (A [r, K], B [N, r], scale)}; FP32 sums with the longest chains that the kernels have: a wave's
    share of the columns, an eighth of them at most, in steps of 4 products, then 16 shares; then the ranks, and the base. Every
    product and sum is off by 2^-24 of the magnitudes' sum at most, the rounding of the operands' parts by as much again."""
    x = np.asarray(x, np.float64)
    m, k = x.shape
    y = np.zeros((m, rows)) if base is None else np.asarray(base, np.float64).copy()
    tol = np.abs(y) * 2.0 ** -24
    for s, (a, b, scale) in pairs.items():
        at = np.nonzero(slot == s)[0]
        if not at.size:
            continue
        a, b, scale = np.asarray(a, np.float64), np.asarray(b, np.float64), np.float64(np.float32(scale))
        y[at] += scale * ((x[at] @ a.T) @ b.T)
        mag = abs(scale) * ((np.abs(x[at]) @ np.abs(a).T) @ np.abs(b).T)
        tol[at] += (k / 8 + 40 + a.shape[0] + 8) * 2.0 ** -24 * mag + 2.0 ** -24 * np.abs(y[at]) + 2.0 ** -120
    return y, tol
