"""Plain forms in 64 bits (numpy) of a mixture-of-experts layer's operators and of the 8-bit products, for their tests."""
import numpy as np

HALF = 2.0 ** -24                    # a rounding to f32 is off by at most this much of the value


def scores(logits, sigmoid):
    l = np.asarray(logits, np.float64)
    l = np.where(np.isnan(l), -np.inf, l)
    if sigmoid:
        return np.where(l >= 0, 1 / (1 + np.exp(-np.abs(l))), np.exp(-np.abs(l)) / (1 + np.exp(-np.abs(l))))
    top = l.max(-1, keepdims=True)
    e = np.exp(l - np.where(np.isfinite(top), top, 0))
    total = e.sum(-1, keepdims=True)
    return e / np.where(total == 0, 1, total)


def route(logits, k, sigmoid=False, renorm=False, scale=1.0, bias=None):
    """(ids, weights) of every token."""
    l = np.asarray(logits, np.float64)
    l = np.where(np.isnan(l), -np.inf, l)
    s = scores(l, sigmoid)
    key = l.copy()
    if bias is not None:
        key = np.where(np.isneginf(l), -np.inf, s + np.asarray(bias, np.float64))
        key = np.where(np.isnan(key), -np.inf, key)
    order = np.argsort(-key, axis=-1, kind="stable")[:, :k]
    ids = np.where(np.isneginf(np.take_along_axis(key, order, -1)), -1, order)
    w = np.where(ids >= 0, np.take_along_axis(s, order, -1), 0.0)
    if renorm:
        if sigmoid:                  # in a form that keeps the ratio of scores that are all tiny
            x = np.where(ids >= 0, np.take_along_axis(l, order, -1), -np.inf)
            m = np.minimum(x, 0).max(-1, keepdims=True)
            w = np.where(ids >= 0, np.exp(np.minimum(x, 0) - np.where(np.isfinite(m), m, 0)) / (1 + np.exp(-np.abs(x))), 0.0)
        total = w.sum(-1, keepdims=True)
        w = w / np.where(total == 0, 1, total)
    return ids.astype(np.int32), scale * w


def sort(ids, E):
    """(row_off, src, slot) by a loop over the assignments."""
    flat = np.asarray(ids).ravel()
    lists = [[] for _ in range(E)]
    for a, e in enumerate(flat):
        if 0 <= e < E:
            lists[e].append(a)
    row_off = np.concatenate([[0], np.cumsum([len(x) for x in lists])]).astype(np.int32)
    src, slot = np.full(flat.size, -1, np.int32), np.full(flat.size, -1, np.int32)
    for r, a in enumerate(a for x in lists for a in x):
        src[r], slot[a] = a, r
    return row_off, src, slot.reshape(np.shape(ids))


def route_grad(logits, ids, dw, sigmoid, renorm, scale):
    """dlogits by the chain rule over the Jacobian of the weights, and the size of the terms that cancel in it."""
    l = np.asarray(logits, np.float64)
    T, E = l.shape
    k = ids.shape[1]
    s = scores(l, sigmoid)
    out, size = np.zeros((T, E)), np.zeros((T, E))
    for t in range(T):
        have = [j for j in range(k) if ids[t, j] >= 0]
        ds = np.zeros((k, E))                        # d s_{ids j} / d l
        for j in have:
            e = ids[t, j]
            if sigmoid:
                ds[j, e] = s[t, e] * (1 - s[t, e])
            else:
                ds[j] = -s[t, e] * s[t]
                ds[j, e] += s[t, e]
        total = sum(s[t, ids[t, j]] for j in have) if renorm and have else 1.0
        sel = np.array([s[t, ids[t, j]] if j in have else 0.0 for j in range(k)])
        for j in have:
            g = scale * float(dw[t, j])
            row = ds[j] / total - (sel[j] / total ** 2 * ds.sum(0) if renorm else 0)
            out[t] += g * row
        p = sel / total
        mean = (p * np.abs(scale * dw[t].astype(np.float64))).sum()
        size[t] = 0 if renorm or sigmoid else s[t] * mean
        for j in have:
            size[t, ids[t, j]] += p[j] * (abs(scale * float(dw[t, j])) + mean)
    return out, size


def quantize(h):
    """(codes, scales) of rows in 64 bits."""
    h = np.asarray(h, np.float64)
    top = np.abs(h).max(-1, initial=0.0)
    with np.errstate(invalid="ignore", over="ignore"):
        scale = (top / 127).astype(np.float32)
    fine = np.isfinite(scale)
    some = fine & (scale >= np.float32(2.0 ** -126))
    step = np.where(some, scale, 1).astype(np.float64)[:, None]
    codes = np.where(some[:, None], np.clip(np.floor(np.where(np.isfinite(h), h, 0) / step + 0.5), -127, 127), 0).astype(np.int8)
    return codes, np.where(fine, np.where(some, scale, 0), np.nan).astype(np.float32)


def act(g, gelu=False):
    g = np.asarray(g, np.float64)
    if gelu:
        return 0.5 * g * (1 + np.tanh(0.7978845608028654 * (g + 0.044715 * g * g * g)))
    return g / (1 + np.exp(-g))


def product(x, xs, w, ws, res=None):
    """(y, bound): the exact value of y and how far f32 may be off it: the sum's rounding and two of the scaling, of the product's
    size; one of the addition, of y's."""
    sums = x.astype(np.int64) @ w.astype(np.int64).T if x.size < 1 << 14 else np.rint(x.astype(np.float64) @ w.astype(np.float64).T)
    y = sums.astype(np.float64) * ws.astype(np.float64) * xs.astype(np.float64)[:, None]
    bound = 3.01 * HALF * np.abs(y)
    if res is not None:
        y = y + res.astype(np.float64)
        bound = bound + 1.01 * HALF * np.abs(y)
    return y, bound + 2.0 ** -148                    # (the smallest f32 values)
