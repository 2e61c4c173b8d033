"""A mixture of experts evaluated in 64 bits with numpy from its definitions
(no code of the backend)."""
import numpy as np

import mxfp4_reference as ref

U = 2.0 ** -24  # half a step of f32, relative


def route(x, top, bias=None, sigmoid=False, groups=1, kept=1, best=1, renorm=True, scale=1.0):
    """ids, weights and what the weights may be off, for rows x [tokens, experts] of any float type."""
    x = np.asarray(x).astype(np.float64)
    tokens, experts = x.shape
    ids = np.full((tokens, top), -1, np.int32)
    weights, off = np.zeros((tokens, top)), np.zeros((tokens, top))
    size = experts // groups
    for t in range(tokens):
        row = np.where(np.isnan(x[t]), -np.inf, x[t])
        with np.errstate(all="ignore"):
            if sigmoid:
                p = 1 / (1 + np.exp(-row))
            else:
                e = np.where(row == row.max(), 1.0, np.exp(row - row.max()))
                e = np.where(row == -np.inf, 0.0, e)
                p = e / e.sum() if e.sum() > 0 else e
            sums = bias is not None or (groups > kept and best == 2)
            c = p + (0 if bias is None else bias.astype(np.float64)) if sums else row
            c = np.where((row > -np.inf) & (c > -np.inf), c, -np.inf)
        if groups > kept:
            values = []
            for g in range(groups):
                s = np.sort(c[g * size:(g + 1) * size])[::-1]
                values.append(s[0] + s[1] if best == 2 and size > 1 and s[1] > -np.inf else s[0])
            order = sorted(range(groups), key=lambda g: (-values[g], g))
            for g in order[kept:]:
                c[g * size:(g + 1) * size] = -np.inf
        order = sorted(range(experts), key=lambda e: (-c[e], e))[:top]
        chosen = [e for e in order if c[e] > -np.inf]
        if not chosen:
            continue
        ids[t, :len(chosen)] = chosen
        y = row[chosen]
        m = y.max() if renorm else row.max()
        with np.errstate(all="ignore"):
            d = np.where(y == m, 0.0, m - y)
            if sigmoid:
                # of the renormalised form's two terms only the second has a rounded difference, and it counts by
                # its share
                m = min(m, 0.0)
                second = np.exp(m - y)
                d = np.where(second > 0, np.abs(m - y) * second / (np.exp(m) + second), 0.0) if renorm else np.zeros(len(y))
                w = 1 / (np.exp(m) + second) if renorm else p[chosen]
            else:
                w = np.exp(-d)
            # the difference's rounding, the exponential's (an ulp), and those of the steps behind it
            each = np.where(w > 0, d, 0) * U + 8 * U
            if renorm:
                total, slack = w.sum(), (w * each).sum() / w.sum() + top * U
            elif sigmoid:
                total, slack = 1.0, 0.0
            else:
                rest = np.where(row == m, 0.0, m - row)
                all_e = np.where(row == -np.inf, 0.0, np.exp(-rest))
                total = all_e.sum()
                slack = (all_e * np.where(all_e > 0, rest, 0)).sum() * U / total + (experts / 16 + 12) * U
        weights[t, :len(chosen)] = scale * w / total
        off[t, :len(chosen)] = np.abs(weights[t, :len(chosen)]) * (each + slack + 4 * U) + 2.0 ** -140
    return ids, weights, off


def order(ids, experts):
    """offsets and order of flat ids."""
    ids = np.asarray(ids).reshape(-1)
    places = [np.flatnonzero(ids == e) for e in range(experts)]
    offsets = np.concatenate([[0], np.cumsum([len(p) for p in places])]).astype(np.int32)
    out = np.full(ids.size, -1, np.int32)
    out[:offsets[-1]] = np.concatenate(places)
    return offsets, out


def product(a, w, bias, act):
    """act(a w^T + bias) of one expert's f64 rows, and what it may be off; act 3 gates columns two by two."""
    if act != 3:
        return ref.product(a, w, bias, act)
    y, off = ref.product(a, w, bias, 0)
    g, dg = ref.product(a, w[0::2], None if bias is None else bias[0::2], 2)
    u, du = y[:, 1::2], off[:, 1::2]
    return g * u, dg * np.abs(u) + (np.abs(g) + dg) * du + U * np.abs(g * u)


def products(a, w, bias, act, offsets, order, gather, scatter, slots):
    """All experts' rows: C (NaN where no place writes) and what it may be off.  a, w: f64 values [rows, k] and
    [experts, n, k]."""
    n = w.shape[1] // 2 if act == 3 else w.shape[1]
    y, off = np.full((slots, n), np.nan), np.full((slots, n), np.nan)
    for e in range(w.shape[0]):
        place = np.arange(offsets[e], offsets[e + 1])
        if not len(place):
            continue
        rows = order[place] // gather if gather else place
        to = order[place] if scatter else place
        y[to], off[to] = product(a[rows], w[e], None if bias is None else bias[e].astype(np.float64), act)
    return y, off


def combine(x, ids, weights, base, experts):
    """The weighted sums in f64, and what f32 sums may be off."""
    tokens, top = ids.shape
    x = x.astype(np.float64).reshape(tokens, top, -1)
    w = np.where((ids >= 0) & (ids < experts), weights.astype(np.float64), 0.0)[..., None]
    real = ((ids >= 0) & (ids < experts))[..., None]
    terms = np.where(real, w * np.where(real, x, 0), 0)
    y, size = terms.sum(1), np.abs(terms).sum(1)
    if base is not None:
        y, size = y + base.astype(np.float64), size + np.abs(base.astype(np.float64))
    return y, (top + 1) * 2 * U * size
