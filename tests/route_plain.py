"""Routing in groups, in 64 bits, expert by expert."""
import numpy as np


def route(x, k, groups=1, top_groups=1, scoring="sigmoid", bias=None, group_top=2, norm=True, scale=1.0):
    """(indices, weights, scores) of float64 logits [T, E]."""
    T, E = x.shape
    idx, w, scores = np.full((T, k), -1), np.zeros((T, k)), np.zeros((T, E))
    size = E // groups
    with np.errstate(all="ignore"):
        for t in range(T):
            l = x[t]
            if scoring == "sigmoid":
                s = np.where(l >= 0, 1 / (1 + np.exp(-l)), np.exp(l) / (1 + np.exp(l)))
            else:
                live = l[l != -np.inf]
                e = np.where(l == -np.inf, 0.0, np.exp(l - (live.max() if live.size else 0.0)))
                s = e / e.sum() if live.size else e
            q = s if bias is None else s + bias
            q = np.where(np.isnan(q), np.inf, q)
            dead = (l == -np.inf) | (q == -np.inf)
            q = np.where(dead, -np.inf, q)
            rank = np.where(dead, -np.inf, np.where(np.isnan(l), np.inf, l)) if bias is None else q
            if top_groups < groups:
                by = rank if bias is None and group_top == 1 else q
                total = []
                for g in range(groups):
                    best = sorted((v for v in by[g * size:(g + 1) * size] if v > -np.inf), reverse=True)[:group_top]
                    total.append(sum(best) if best else -np.inf)
                kept = sorted(range(groups), key=lambda g: (-total[g], g))[:top_groups]
                rank = np.array([rank[e] if e // size in kept else -np.inf for e in range(E)])
            order = sorted((e for e in range(E) if rank[e] > -np.inf), key=lambda e: (-rank[e], e))[:k]
            idx[t, :len(order)] = order
            p = s[order]
            w[t, :len(order)] = scale * (p / (p.sum() + 1e-20) if norm else p)
            scores[t] = s
    return idx, w, scores


def gradient(x, idx, dw, scoring, norm, scale, scores):
    """dlogits in float64 for weights' gradients dw."""
    dl = np.zeros_like(x)
    for t in range(x.shape[0]):
        on = idx[t] >= 0
        i, s, d = idx[t][on], scores[t][idx[t][on]], scale * dw[t][on]
        S = s.sum() + 1e-20
        ds = (d - (d * s / S).sum()) / S if norm else d
        if scoring == "sigmoid":
            dl[t, i] = ds * s * (1 - s)
        else:
            dl[t, i] = ds * s
            if not norm:
                dl[t] -= scores[t] * (ds * s).sum()
    return dl
