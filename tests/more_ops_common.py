"""Plain 64-bit forms of sorted rows, their gradients, the routing weights' gradient and 8-bit rows, on the host."""
import numpy as np


def sort(x, inv, w, xs):
    """xs with row inv[t][k] = (w[t][k]) x[t]; the others as they were."""
    out = xs.copy()
    for t in range(inv.shape[0]):
        for k, r in enumerate(inv[t]):
            if 0 <= r < len(out):
                out[r] = x[t] if w is None else w[t, k] * x[t]
    return out


def gathered(rows, inv):
    """rows[inv], zeros where an entry names none: [T][n_used][D]."""
    there = (inv >= 0) & (inv < len(rows))
    return np.where(there[..., None], rows[np.where(there, inv, 0)], 0.0) if len(rows) else np.zeros(inv.shape + rows.shape[1:])


def weights_by_logits(l, ids, score, renorm, scale):
    """The routing's weights [T][n_used] as a function of the logits [T][E], the experts held fixed: ids outside 0 .. E - 1 have none, experts whose
    logit is -infinity take no part."""
    E = l.shape[1]
    there = (ids >= 0) & (ids < E)
    lc = np.where(there, np.take_along_axis(l, np.where(there, ids, 0), 1), -np.inf)
    with np.errstate(over="ignore", invalid="ignore", divide="ignore"):
        if score == "softmax":
            if renorm:
                e = np.exp(lc - lc.max(1, keepdims=True))
                w = e / e.sum(1, keepdims=True)
            else:
                top = l.max(1, keepdims=True)
                w = np.exp(lc - top) / np.exp(l - top).sum(1, keepdims=True)
        else:
            ls = -np.logaddexp(0, -lc)
            if renorm:
                e = np.exp(ls - ls.max(1, keepdims=True))
                w = e / e.sum(1, keepdims=True)
            else:
                w = np.exp(ls)
    return np.where(np.isnan(w), 0.0, w) * scale


def route_grad(l, ids, dw, score, renorm, scale):
    """dlogits [T][E], and for each a size that its roundings are relative to."""
    T, E = l.shape
    out, size = np.zeros((T, E)), np.zeros((T, E))
    for t in range(T):
        chosen = [(e, dw[t, k]) for k, e in enumerate(ids[t]) if 0 <= e < E and l[t, e] > -np.inf]
        if not chosen:
            continue
        e, d = np.array([c[0] for c in chosen]), np.array([c[1] for c in chosen], np.float64)
        lc = l[t, e]
        if score == "softmax":
            if renorm:
                p = np.exp(lc - lc.max())
                p /= p.sum()
                m = (p * d).sum()
                out[t, e], size[t, e] = p * (d - m), p * (np.abs(d) + (p * np.abs(d)).sum())
            else:
                p = np.exp(l[t] - l[t].max())
                p /= p.sum()
                m, a = (p[e] * d).sum(), (p[e] * np.abs(d)).sum()
                out[t], size[t] = -p * m, p * a
                out[t, e] += p[e] * d
                size[t, e] += p[e] * np.abs(d)
        else:
            ls = -np.logaddexp(0, -lc)
            rest = np.exp(-np.logaddexp(0, lc))
            if renorm:
                p = np.exp(ls - ls.max())
                p /= p.sum()
                m = (p * d).sum()
                out[t, e], size[t, e] = p * rest * (d - m), p * rest * (np.abs(d) + (p * np.abs(d)).sum())
            else:
                out[t, e] = np.exp(ls) * rest * d
                size[t, e] = np.abs(out[t, e])
    return out * scale, size * abs(scale)


def quantize(x):
    """Codes [R][K] and f32 scales [R] of rows x (numbers that f32 holds)."""
    x = np.asarray(x, np.float64)
    top = np.abs(x).max(1)
    bad = ~np.isfinite(top)
    safe = np.where(bad | (top == 0), 1.0, top)
    # 127 x is exact, and the quotient's rounding makes no border between two codes of what is none.
    codes = np.rint(127 * np.where(bad[:, None], 0.0, x) / safe[:, None])
    scales = np.where(bad, 0.0, top).astype(np.float32) / np.float32(127)
    return codes.astype(np.int8), np.where(bad, np.float32(np.nan), scales).astype(np.float32)


def product(codes, scales, wc, ws, offsets, rows):
    """f32 results [rows][N], rounded as the framework says: the exact sum, the row's scale, the matrix's row's; and which rows have an expert."""
    out, named = np.zeros((rows, wc.shape[1]), np.float32), np.zeros(rows, bool)
    for e in range(wc.shape[0]):
        a, b = offsets[e], min(offsets[e + 1], rows)
        if b > a:
            acc = (codes[a:b].astype(np.float64) @ wc[e].astype(np.float64).T).astype(np.float32)
            with np.errstate(over="ignore", invalid="ignore", under="ignore"):
                out[a:b] = acc * scales[a:b, None] * ws[e][None]
            named[a:b] = True
    return out, named
