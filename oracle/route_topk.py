"""Expert choice from router logits in 64 bits, row by row (``gpu.routing.route_topk``).

Choice values that are equal in 64 bits go by the larger logit, then by the
lower index; groups of equal worth by the logit of their best expert, then by
the lower index."""
import numpy as np


def route_topk(logits, k, score="softmax", bias=None, n_group=1, topk_group=1, group_score="max", renormalize=True,
               scale=1.0):
    """``logits`` (T, E) as exact float64 values; returns (weights float64, ids int64)."""
    l = np.asarray(logits, np.float64)
    T, E = l.shape
    b = np.zeros(E) if bias is None else np.asarray(bias, np.float64)
    W, I = np.zeros((T, k)), np.full((T, k), E, np.int64)
    for t in range(T):
        row = l[t]
        if np.isnan(row).any() or (score == "softmax" and np.isposinf(row).any()):
            W[t], I[t] = np.nan, np.arange(k)
            continue
        masked = np.isneginf(row)
        if score == "softmax":
            p = np.exp(row - row.max()) if not masked.all() else np.zeros(E)
            s = p / p.sum() if not masked.all() else p
        else:
            with np.errstate(over="ignore"):
                s = 1.0 / (1.0 + np.exp(-row))
        if bias is None and not (n_group > 1 and topk_group < n_group and group_score == "top2"):
            c = row.copy()             # same order as the scores, without their rounding
        else:
            c = np.where(masked, -np.inf, s + b)
        if np.isnan(c).any():
            W[t], I[t] = np.nan, np.arange(k)
            continue
        if n_group > 1:
            g = c.reshape(n_group, -1)
            worth, lead = [], []
            for v, r in zip(g, row.reshape(n_group, -1)):
                lead.append(r[v == v.max()].max())
                v = np.sort(v)[::-1]
                second = v[1] if len(v) > 1 and v[1] > -np.inf else 0.0
                worth.append(v[0] + second if group_score == "top2" else v[0])
            keep = sorted(range(n_group), key=lambda i: (-worth[i], -lead[i], i))[:topk_group]
            for i in range(n_group):
                if i not in keep:
                    c[i * (E // n_group):(i + 1) * (E // n_group)] = -np.inf
        order = [e for e in sorted(range(E), key=lambda e: (-c[e], -row[e], e)) if c[e] > -np.inf][:k]
        w = s[order]
        if renormalize:
            w = w / w.sum() if w.sum() > 0 else np.zeros_like(w)
        W[t, : len(order)], I[t, : len(order)] = w * scale, order
    return W, I
