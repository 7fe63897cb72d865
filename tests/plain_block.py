"""Plain 64-bit forms of the operators of a block in plain rows."""
import math

import numpy as np

E4M3 = np.sort(np.concatenate([np.arange(8) * 2.0 ** -9] + [(8 + np.arange(8)) * 2.0 ** (e - 10) for e in range(1, 16)]))
E4M3 = E4M3[E4M3 <= 448.0]  # 0 .. 448: the last of the top binade is NaN's code


def e4m3_round(q):
    """The nearest e4m3 values, halves to even (the last mantissa bit of the value)."""
    a = np.minimum(np.abs(q), 448.0)
    hi = np.clip(np.searchsorted(E4M3, a), 1, len(E4M3) - 1)
    lo = hi - 1
    middle = (E4M3[lo] + E4M3[hi]) / 2
    at = np.where(a < middle, lo, np.where(a > middle, hi, np.where(lo % 2 == 0, lo, hi)))
    return np.copysign(E4M3[at], q)


def e4m3_decode(codes):
    c = np.asarray(codes, np.uint8).astype(int)
    e, m = c >> 3 & 15, c & 7
    v = np.where(e == 0, m * 2.0 ** -9, (8 + m) * 2.0 ** (e - 10.0))
    v = np.where((c & 127) == 127, np.nan, v)
    return np.where(c & 128, -v, v)


def packed(v, codes, scale_columns):
    """(code values, scales) of the rows of v, whose values are fp32's."""
    v = np.asarray(v, np.float64)
    R, C = v.shape
    B = scale_columns or C
    n = -(-C // B)
    top = 127.0 if codes == "int8" else 448.0
    q, scales = np.zeros_like(v), np.zeros((R, n))
    for b in range(n):
        part = v[:, b * B:(b + 1) * B]
        most = np.abs(part).max(axis=1)
        # (a NaN or an infinity among the block's: all of it reads back as NaN)
        with np.errstate(invalid="ignore", over="ignore"):
            s = np.where(np.isfinite(most), (most / top).astype(np.float32).astype(np.float64), np.nan)
        by = np.where(s > 0, s, 1.0)[:, None]
        with np.errstate(invalid="ignore", over="ignore"):
            x = np.where(np.isfinite(part), part, 0.0) / by
            if codes == "int8":
                x = np.copysign(np.minimum(np.floor(np.abs(x) + 0.5), 127.0), x)
            else:
                x = e4m3_round(np.clip(x.astype(np.float32).astype(np.float64), -448, 448))
        q[:, b * B:(b + 1) * B] = np.where((s > 0)[:, None], x, 0.0)
        scales[:, b] = s
    return q, scales


def unpacked(q, scales, scale_columns):
    B = scale_columns or q.shape[1]
    return q * np.repeat(scales, B, axis=1)[:, :q.shape[1]]


def norm(s, w, epsilon):
    """(y, 1 / rms) of the rows of s."""
    r = 1 / np.sqrt((s * s).mean(axis=1, keepdims=True) + epsilon)
    return s * r * (1.0 if w is None else w), r


def norm_gradient(dy, s, w, ds, epsilon):
    """(dx, dw, the sizes of dx's terms, the sizes of dw's)."""
    r = 1 / np.sqrt((s * s).mean(axis=1, keepdims=True) + epsilon)
    n, g = s * r, dy * (1.0 if w is None else w)
    dx = r * (g - n * (g * n).mean(axis=1, keepdims=True))
    size = r * (np.abs(g) + np.abs(n) * np.abs(g * n).mean(axis=1, keepdims=True))
    if ds is not None:
        dx, size = dx + ds, size + np.abs(ds)
    return dx, (dy * n).sum(axis=0), size, np.abs(dy * n).sum(axis=0)


_erfc = np.vectorize(math.erfc, otypes=[np.float64])


def logistic(z):
    with np.errstate(over="ignore"):
        e = np.exp(-np.abs(z))
    return np.where(z >= 0, 1.0, e) / (1 + e)


def activation(z, name):
    """(act(z), act'(z), the sizes of act' 's terms)."""
    z = np.asarray(z, np.float64)
    if name == "none":
        return z, np.ones_like(z), np.ones_like(z)
    if name == "relu":
        d = (z > 0).astype(np.float64)
        return np.where(z <= 0, 0.0, z), d, d
    if name == "silu":
        s = logistic(z)
        return z * s, s + z * s * (1 - s), s + np.abs(z) * s * (1 - s)
    if name == "gelu":
        c, p = 0.5 * _erfc(-z * math.sqrt(0.5)), np.exp(-z * z / 2) / math.sqrt(2 * math.pi)
        return z * c, c + z * p, c + np.abs(z) * p
    k = 2 * math.sqrt(2 / math.pi)
    s = logistic(k * (z + 0.044715 * z ** 3))
    d = k * (1 + 3 * 0.044715 * z * z)
    return z * s, s + z * s * (1 - s) * d, s + np.abs(z) * s * (1 - s) * d


def gated(gate, up, name, limit):
    """(a, c, y) of a gated activation and the gradients' factors (da, dc)."""
    L = limit or np.inf
    a, da, size = activation(np.minimum(gate, L), name)
    c = np.ones_like(gate) if up is None else np.clip(up, -L, L)
    dc = np.zeros_like(gate) if up is None else (np.abs(up) <= L).astype(np.float64)
    return a, c, da * (gate <= L), dc, size


def scores(l, kind):
    if kind == "sigmoid":
        return logistic(l)
    m = l.max(axis=1, keepdims=True)
    with np.errstate(invalid="ignore"):
        e = np.exp(l - np.where(np.isneginf(m), 0.0, m))
        t = e.sum(axis=1, keepdims=True)
    return e / np.where(t == 0, 1.0, t)


def route(l, biases, k, kind, groups=1, chosen_groups=1, best=1, renormalize=True, scale=1.0):
    """(chosen, gates): experts in order of s + b (of l without b), ties by index, -inf last."""
    T, E = l.shape
    s = scores(l, kind)
    out = np.isneginf(l) | np.isnan(l)
    key = l if biases is None else s + biases
    if groups > 1:
        of = (s if biases is None and best == 2 else key).reshape(T, groups, E // groups)
        of = -np.sort(-np.where(out.reshape(of.shape), -np.inf, of), axis=2)[:, :, :best]
        total = np.where(np.isneginf(of), 0.0, of).sum(axis=2)
        total = np.where(np.isneginf(of[:, :, 0]), -np.inf, total)
        order = np.argsort(-total, axis=1, kind="stable")[:, :chosen_groups]
        inside = np.zeros((T, groups), bool)
        np.put_along_axis(inside, order, True, axis=1)
        inside = np.repeat(inside, E // groups, axis=1)
    else:
        inside = np.ones((T, E), bool)
    chosen = np.zeros((T, k), int)
    for t in range(T):
        order = sorted((e for e in range(E) if inside[t, e]), key=lambda e: (out[t, e], 0.0 if out[t, e] else -key[t, e], e))
        chosen[t] = order[:k]
    return chosen, scale * (shares(l, chosen, kind) if renormalize else np.take_along_axis(s, chosen, axis=1))


def shares(l, chosen, kind):
    """s_j / the sum of the chosen s, by the scores' logarithms: the quotient also where the scores
    themselves are too small for a number.  Nothing but -inf: 0."""
    m = np.take_along_axis(l, chosen, axis=1)
    if kind == "sigmoid":
        with np.errstate(over="ignore"):
            m = np.minimum(m, 0) - np.log1p(np.exp(-np.abs(m)))
    top = m.max(axis=1, keepdims=True)
    e = np.exp(m - np.where(np.isneginf(top), 0.0, top))
    total = e.sum(axis=1, keepdims=True)
    return e / np.where(total == 0, 1.0, total)


def route_gradient(l, chosen, dg, kind, renormalize, scale):
    """(the logits' gradients, the sizes of their terms)."""
    T, E = l.shape
    s = scores(l, kind)
    out, size = np.zeros((T, E)), np.zeros((T, E))
    for t in range(T):
        at = [j for j, e in enumerate(chosen[t]) if 0 <= e < E]
        if not at:
            continue
        c, d = np.asarray(chosen[t])[at].astype(int), scale * dg[t, at]
        if renormalize:
            # gate_i = s_i / S: its derivative by log s_j is gate_i ([i = j] - gate_j); log s by l is 1 (a
            # softmax's common sum cancels) or 1 - s
            p = shares(l[t:t + 1], c[None], kind)[0]
            by, sizes = p * (d - (p * d).sum()), p * (np.abs(d) + (p * np.abs(d)).sum())
        else:
            by, sizes = s[t, c] * d, s[t, c] * np.abs(d)
        if kind == "sigmoid":
            by, sizes = by * logistic(-l[t, c]), sizes * logistic(-l[t, c])
        np.add.at(out[t], c, by)
        np.add.at(size[t], c, sizes)
        if kind == "softmax" and not renormalize:
            out[t] -= s[t] * by.sum()
            size[t] += s[t] * sizes.sum()
    return out, size


def lists(chosen, experts):
    """(offsets, rows, places) in expert order."""
    T, k = chosen.shape
    flat = chosen.reshape(-1)
    order = np.argsort(flat, kind="stable")
    places = np.empty(T * k, int)
    places[order] = np.arange(T * k)
    offsets = np.concatenate([[0], np.cumsum(np.bincount(flat, minlength=experts))])
    return offsets, order // k, places.reshape(T, k)
