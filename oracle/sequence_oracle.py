"""Float64 restatements of embeddings, gated recurrences along sequences and sampling of tokens, from their formulas.  Matrices are (rows,
columns) arrays, a column is a token."""
import math

import numpy as np

from oracle.token_oracle import is_token


# ---- embeddings

def embed(table, labels, mult=1.0):
    table, l = np.asarray(table, dtype=np.float64), np.asarray(labels, dtype=np.float64).reshape(-1)
    out = np.zeros((table.shape[0], l.size))
    for c in np.flatnonzero(is_token(l, table.shape[1])):
        out[:, c] = mult * table[:, int(l[c])]
    return out


def embed_grad(dy, labels, vocab, mult=1.0):
    """(gradient, the same sums of magnitudes, number of columns of each token)."""
    dy, l = np.asarray(dy, dtype=np.float64), np.asarray(labels, dtype=np.float64).reshape(-1)
    g, a, n = np.zeros((dy.shape[0], vocab)), np.zeros((dy.shape[0], vocab)), np.zeros(vocab)
    for c in np.flatnonzero(is_token(l, vocab)):
        g[:, int(l[c])] += dy[:, c]
        a[:, int(l[c])] += np.abs(dy[:, c])
        n[int(l[c])] += 1
    return mult * g, abs(mult) * a, n


# ---- gated recurrences

def gates(pre):
    """a = sigmoid(g), 1 - a, u."""
    pre = np.asarray(pre, dtype=np.float64)
    f = pre.shape[0] // 2
    with np.errstate(over='ignore'):
        return 1.0 / (1.0 + np.exp(-pre[:f])), 1.0 / (1.0 + np.exp(pre[:f])), pre[f:]


def borders(cols, offsets=None, sequences=1):
    if offsets is not None:
        return [int(o) for o in np.asarray(offsets).reshape(-1)]
    return [q * (cols // sequences) for q in range(sequences + 1)]


def gated_scan(pre, at, state=None):
    """(columns, last columns, and how far a result may be off in units of the rounding of one operation: every step adds a few to what
    the last one had, of the magnitudes that it handles; both for columns and for last columns).  Columns of no sequence are NaN."""
    a, s, u = gates(pre)
    f, n = u.shape[0], len(at) - 1
    y, last = np.full(u.shape, np.nan), np.zeros((f, n)) if state is None else np.array(state, dtype=np.float64)
    off, last_off = np.zeros(u.shape), np.zeros((f, n))
    with np.errstate(invalid='ignore', over='ignore'):
        for q in range(n):
            h = last[:, q].copy()
            m, e = np.abs(h), np.zeros(f)
            for c in range(at[q], at[q + 1]):
                h = a[:, c] * h + s[:, c] * u[:, c]
                m = a[:, c] * m + s[:, c] * np.abs(u[:, c])
                e = a[:, c] * e + m
                y[:, c], off[:, c] = h, e
            last[:, q], last_off[:, q] = h, e
    return y, last, off, last_off


def gated_scan_grad(dy, pre, out, at, state=None, last_deriv=None):
    """Derivatives by pre and by state, and the bounds as above.  Columns of no sequence are NaN."""
    a, s, u = gates(pre)
    dy, out = np.asarray(dy, dtype=np.float64), np.asarray(out, dtype=np.float64)
    f, n = u.shape[0], len(at) - 1
    dpre, off = np.full((2 * f, u.shape[1]), np.nan), np.zeros((2 * f, u.shape[1]))
    dstate = np.zeros((f, n)) if last_deriv is None else np.array(last_deriv, dtype=np.float64)
    state_off = np.zeros((f, n))
    for q in range(n):
        back = dstate[:, q].copy()
        m, e = np.abs(back), np.zeros(f)
        for c in range(at[q + 1] - 1, at[q] - 1, -1):
            h = out[:, c - 1] if c > at[q] else np.zeros(f) if state is None else np.asarray(state, dtype=np.float64)[:, q]
            both, m = dy[:, c] + back, np.abs(dy[:, c]) + m
            e = e + m
            dpre[:f, c], dpre[f:, c] = a[:, c] * s[:, c] * (h - u[:, c]) * both, s[:, c] * both
            off[f:, c] = s[:, c] * e
            off[:f, c] = a[:, c] * s[:, c] * ((np.abs(h) + np.abs(u[:, c])) * np.abs(both) + np.abs(h - u[:, c]) * e)
            back, m, e = a[:, c] * both, a[:, c] * m, a[:, c] * (e + m)
        dstate[:, q], state_off[:, q] = back, e
    return dpre, dstate, off, state_off


# ---- sampling

def sample_token(x, uniform, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, part=1.0):
    """(token, log probability, the kept entries) of one column.  part: a factor of what top_p asks for."""
    x = np.asarray(x, dtype=np.float32).astype(np.float64)
    temperature, top_k, top_p, min_p, u = (float(np.float32(v)) for v in (temperature, top_k, top_p, min_p, uniform))
    h = x.size
    if h == 0 or (np.isnan(x) | (x == np.inf)).any():
        return -1, math.nan if h else 0.0, []
    best = int(np.argmax(x))
    if x[best] == -np.inf:
        return -1, 0.0, []
    if not temperature > 0:
        return best, 0.0, [best]
    with np.errstate(invalid='ignore', over='ignore'):
        w = np.where(x == -np.inf, 0.0, np.exp((x - x[best]) / temperature))
    kept = sorted(range(h), key=lambda i: (-x[i], i))
    if 1 <= top_k < h:
        kept = kept[:int(top_k)]
    if min_p > 0:
        kept = [i for i in kept if w[i] >= min(min_p, 1.0)]
    if top_p < 1:
        total, up_to, n = math.fsum(w[i] for i in kept), 0.0, 0
        while n == 0 or (n < len(kept) and up_to < part * top_p * total):
            up_to += w[kept[n]]
            n += 1
        kept = kept[:n]
    kept = sorted(i for i in kept if w[i] > 2.0 ** -46)
    total, up_to = math.fsum(w[i] for i in kept), 0.0
    u = min(max(u, 0.0), 1.0) if u == u else 0.0
    for i in kept:
        up_to += w[i]
        if up_to > u * total:
            break
    return i, math.log(w[i] / total), kept
