"""The routing operators' definitions in FP64 on the CPU (numpy), for the tests."""
import numpy as np


def softmax(x):
    top = x.max(1, keepdims=True)
    top = np.where(np.isneginf(top), 0.0, top)
    e = np.exp(x - top)
    total = e.sum(1, keepdims=True)
    return np.divide(e, total, out=np.zeros_like(e), where=total > 0)


def scores(x, score):
    with np.errstate(over="ignore"):
        return softmax(x) if score == "softmax" else 1.0 / (1.0 + np.exp(-x))


def route(x, top_k, score="softmax", bias=None, groups=1, top_groups=1, group_score="max", renormalize=True, scale=1.0):
    """One row at a time, one choice at a time: the largest eligible choice value, the lowest index on ties."""
    x = np.asarray(x, np.float64)
    n, experts = x.shape
    s = scores(x, score)
    c = s if bias is None else s + np.asarray(bias, np.float64)
    c = np.where(np.isneginf(x), -np.inf, c)
    ids = np.full((n, top_k), -1, np.int32)
    w = np.zeros((n, top_k))
    per = experts // groups
    for t in range(n):
        row = c[t].copy()
        if groups > 1:
            worth = []
            for g in range(groups):
                best = sorted((v for v in row[g * per:(g + 1) * per] if v > -np.inf), reverse=True)
                worth.append(-np.inf if not best else best[0] if group_score == "max" else sum(best[:2]))
            order = sorted(range(groups), key=lambda g: (-worth[g], g))
            for g in order[top_groups:]:
                row[g * per:(g + 1) * per] = -np.inf
        for i in range(top_k):
            j = int(np.argmax(row))
            if row[j] == -np.inf:
                break
            ids[t, i] = j
            w[t, i] = s[t, j]
            row[j] = -np.inf
        if renormalize and w[t].sum() > 0:
            w[t] /= w[t].sum()
    return ids, w * scale


def route_grad(g, x, ids, score="softmax", renormalize=True, scale=1.0):
    """Jacobians written out: d weights / d scores, then d scores / d logits."""
    x = np.asarray(x, np.float64)
    s = scores(x, score)
    out = np.zeros_like(x)
    for t in range(x.shape[0]):
        slots = [(i, j) for i, j in enumerate(ids[t]) if 0 <= j < x.shape[1]]
        total = sum(s[t, j] for _, j in slots)
        ds = np.zeros(x.shape[1])
        for i, j in slots:
            gi = float(g[t, i]) * scale
            if renormalize:
                if total > 0:
                    ds[j] += gi / total
                    for _, q in slots:
                        ds[q] -= gi * s[t, j] / total ** 2
            else:
                ds[j] += gi
        if score == "sigmoid":
            out[t] = ds * s[t] * (1 - s[t])
        else:
            out[t] = s[t] * (ds - (ds * s[t]).sum())
    return out


def plan(ids, experts):
    flat = np.asarray(ids).reshape(-1)
    lists = [[q for q in range(flat.size) if flat[q] == e] for e in range(experts)] if flat.size < 3000 else \
        [np.flatnonzero(flat == e).tolist() for e in range(experts)]
    offsets = np.concatenate([[0], np.cumsum([len(v) for v in lists])]).astype(np.int32)
    order = np.full(flat.size, -1, np.int32)
    pos = np.full(flat.size, -1, np.int32)
    rows = [q for v in lists for q in v]
    order[:len(rows)] = rows
    pos[rows] = np.arange(len(rows))
    return offsets, order, pos.reshape(np.asarray(ids).shape)


def gathered(x, order, top_k):
    out = np.zeros((order.size, x.shape[1]))
    kept = order >= 0
    out[kept] = x[order[kept] // top_k]
    return out


def gemm(xs, w, offsets):
    out = np.zeros((xs.shape[0], w.shape[1]))
    for e in range(w.shape[0]):
        out[offsets[e]:offsets[e + 1]] = xs[offsets[e]:offsets[e + 1]] @ w[e].T
    return out


def gemm_grad_w(g, xs, offsets):
    return np.stack([g[a:b].T @ xs[a:b] for a, b in zip(offsets[:-1], offsets[1:])])


def combine(y, pos, weights):
    out = np.zeros((pos.shape[0], y.shape[1]))
    for s in range(pos.shape[1]):
        kept = pos[:, s] >= 0
        out[kept] += (weights[kept, s, None] if weights is not None else 1.0) * y[pos[kept, s]]
    return out


def combine_grad(g, y, pos, weights):
    dy = np.zeros_like(y)
    dw = np.zeros(pos.shape)
    for s in range(pos.shape[1]):
        kept = pos[:, s] >= 0
        dy[pos[kept, s]] = (weights[kept, s, None] if weights is not None else 1.0) * g[kept]
        dw[kept, s] = (g[kept] * y[pos[kept, s]]).sum(1)
    return dy, dw
