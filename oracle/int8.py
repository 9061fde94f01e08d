"""Float64 restatement of the int8 operators and of the expert choice (numpy), with error bounds."""
import numpy as np

LEAST = 127.0 * 2.0 ** -100
U32 = 2.0 ** -24                # half a step of fp32, relative


def quantise(v):
    """float64 rows -> (whole numbers, fp32 scales (rows, 1)); rows that are not finite: zeros and NaN."""
    v = np.asarray(v, np.float64)
    real = np.isfinite(v).all(-1, keepdims=True)
    a = np.maximum(np.where(real, np.abs(np.where(np.isfinite(v), v, 0.0)), 0.0).max(-1, keepdims=True), LEAST)
    q = np.round(np.where(real, v, 0.0) * 127.0 / a)
    return q, np.where(real, (a / 127.0).astype(np.float32), np.float32(np.nan))


def silu_mul(gate, up):
    with np.errstate(all="ignore"):
        far = gate < -700
        mid = np.exp(np.where(far, gate / 2, 0.0))
        return np.where(far, (gate * mid) * (mid * up), gate / (1.0 + np.exp(-np.where(far, 0.0, gate))) * up)


def product(q, xs, w, ws, bias=None):
    """Rows (M, K) of whole numbers with scales (M, 1) times weights (N, K) with scales (N,): (values, how far fp32
    arithmetic may be off). The sum is exact; it is rounded to fp32, the scales' product is, the product of the two
    is, and the sum with the bias is."""
    y = (q.astype(np.float64) @ w.astype(np.float64).T) * xs.astype(np.float64) * ws.astype(np.float64)
    tol = np.abs(y) * 3 * U32
    if bias is not None:
        y = y + bias
        tol = tol + (np.abs(y) + tol) * U32
    return y, tol * (1 + 8 * U32) + 2.0 ** -148


def expert(q, xs, w13, s13, w2, s2):
    """Rows of one expert through its two products: (y, how far it may be off). A value of h next to a border between
    two whole numbers may fall on either side of it: it counts with a step."""
    inter = w13.shape[0] // 2
    gu, _ = product(q, xs, w13, s13)
    g, u = gu[:, :inter], gu[:, inter:]
    h = silu_mul(g, u)
    # gate and up are off by 3 roundings each, silu's slope is at most 1 + |g| in relative terms; exponential (2 steps:
    # 4 roundings), its sum with one, quotient and product 3 more
    rel = (3 * (1 + np.abs(g)) + 3 + 8) * U32
    hq, hs = quantise(h)
    a = hs.astype(np.float64) * 127.0
    # the row's scale: as far off as its largest value may be
    top = np.abs(h).argmax(-1)
    rel_a = np.maximum(np.take_along_axis(rel, top[:, None], 1), (np.abs(h) * (1 + rel) / a - 1).max(-1, keepdims=True)) + U32
    t = np.abs(h) * 127.0 / a
    off = t * (rel + rel_a + 4 * U32)
    border = np.abs(t - np.floor(t) - 0.5) <= off
    y, tol = product(hq, hs, w2, s2)
    tol = tol + np.abs(y) * rel_a
    tol = tol + (border.astype(np.float64) @ np.abs(w2.astype(np.float64)).T) * hs.astype(np.float64) * s2.astype(np.float64)
    return y, tol


def layer(q, xs, w13, s13, w2, s2, tw, ids, expert_map=None, rows16=False):
    """(out, how far fp32 arithmetic may be off); ids without a local expert contribute nothing. rows16: for slots'
    rows that are rounded to fp16 before the sum (no schedule of the layer does so), times a power of two that puts the largest of 32 columns into [2^14, 2^15):
    off by 2^-11 of a value, and by 2^-25 (half of fp16's least step) of 2^-14 of that largest one."""
    T, k = ids.shape
    out, tol = np.zeros((T, w2.shape[1])), np.zeros((T, w2.shape[1]))
    size = np.zeros_like(out)
    local = ids if expert_map is None else np.where((ids >= 0) & (ids < len(expert_map)),
                                                    np.asarray(expert_map)[np.clip(ids, 0, len(expert_map) - 1)], -1)
    for e in range(w13.shape[0]):
        t, j = np.nonzero(local == e)
        if len(t) == 0:
            continue
        y, d = expert(q[t], xs[t], w13[e], s13[e], w2[e], s2[e])
        if rows16:
            block = np.abs(y).reshape(len(t), -1, 32).max(-1).repeat(32, axis=1)
            d = d + (np.abs(y) + d) * 2.0 ** -11 + block * 2.0 ** -39
        w = tw[t, j].astype(np.float64)[:, None]
        np.add.at(out, t, y * w)
        np.add.at(tol, t, d * np.abs(w))
        np.add.at(size, t, np.abs(y * w))
    return out, tol + size * (k + 1) * U32


def route(logits, top_k, scoring, bias, groups, top_groups, renorm, scale):
    """(weights, ids), one token and one pick at a time."""
    T, E = logits.shape
    w, ids = np.zeros((T, top_k)), np.full((T, top_k), -1, np.int32)
    for t in range(T):
        l = np.where(np.isnan(logits[t]), -np.inf, np.minimum(logits[t].astype(np.float64), np.finfo(np.float32).max))
        live = l > -np.inf
        with np.errstate(all="ignore"):
            if scoring == "sigmoid":
                p = 1.0 / (1.0 + np.exp(-l))
            else:
                x = np.exp(l - (l.max() if live.any() else 0.0))
                p = x / x.sum()
            c = p + (0.0 if bias is None else bias.astype(np.float64))
            # without a bias both scores grow with the logit, also where they underflow or reach one
            order = l if bias is None else c
        order = np.where(live & (c > -np.inf), order, -np.inf)
        if groups > 1:
            size = E // groups
            score = []
            for g in range(groups):
                part = np.sort(order[g * size:(g + 1) * size])[::-1]
                two = bias is not None and size > 1 and part[1] > -np.inf
                score.append(part[0] + part[1] if two else part[0])
            stay = sorted(range(groups), key=lambda g: (-score[g], g))[:top_groups]
            order = np.where(np.isin(np.arange(E) // size, stay), order, -np.inf)
        best = [e for e in sorted(range(E), key=lambda e: (-order[e], e)) if order[e] > -np.inf][:top_k]
        ids[t, :len(best)] = best
        v = p[best]
        if renorm and len(best):
            v = v / v.sum() if v.sum() > 0 else np.zeros_like(v)
        w[t, :len(best)] = v * scale
    return w, ids
