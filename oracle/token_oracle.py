"""Float64 restatements of the operators on columns of tokens: layer norm, gated products, dropout by a counter-based
generator, log probabilities of tokens; forward and backward, from their formulas.  Matrices are (rows, columns) arrays, a
column is a case."""
import math

import numpy as np

try:
    from scipy.special import erfc as _erfc
except ImportError:                                     # (scipy is there wherever the tests run)
    _erfc = np.vectorize(math.erfc)


def _vec(v, h, default):
    return np.full((h, 1), default) if v is None else np.asarray(v, dtype=np.float64).reshape(h, 1)


# ---- layer norm

def normalised(x, eps):
    """(x^, 1 / std) of every column."""
    x = np.asarray(x, dtype=np.float64)
    d = x - x.mean(axis=0, keepdims=True)
    r = 1.0 / np.sqrt((d * d).mean(axis=0, keepdims=True) + float(np.float32(eps)))
    return d * r, r


def layer_norm(x, gain=None, bias=None, eps=1e-5):
    h = np.shape(x)[0]
    return _vec(gain, h, 1.0) * normalised(x, eps)[0] + _vec(bias, h, 0.0)


def layer_norm_grad(dy, x, gain=None, eps=1e-5):
    """Derivatives by x, gain and bias (the sums over the columns)."""
    xh, r = normalised(x, eps)
    dy = np.asarray(dy, dtype=np.float64)
    g = dy * _vec(gain, dy.shape[0], 1.0)
    dx = r * (g - g.mean(axis=0, keepdims=True) - xh * (g * xh).mean(axis=0, keepdims=True))
    return dx, (dy * xh).sum(axis=1, keepdims=True), dy.sum(axis=1, keepdims=True)


# ---- gated products

def gate(act, g):
    """(activation, slope)."""
    g = np.asarray(g, dtype=np.float64)
    if act in (None, 'linear'):
        return g, np.ones_like(g)
    if act == 'relu':
        return np.maximum(g, 0.0), (g > 0).astype(np.float64)
    if act == 'tanh':
        return np.tanh(g), 1.0 / np.cosh(np.clip(g, -300, 300)) ** 2
    if act == 'gelu':
        phi = 0.5 * _erfc(-g / math.sqrt(2.0))
        return g * phi, phi + g * np.exp(-0.5 * g * g) / math.sqrt(2.0 * math.pi)
    with np.errstate(over='ignore'):
        s, c = 1.0 / (1.0 + np.exp(-g)), 1.0 / (1.0 + np.exp(g))
    return (s, s * c) if act == 'sigmoid' else (g * s, s + g * s * c)


def dot_gated(m1, m2, bias=None, act='silu'):
    """(act(P[:f]) * P[f:], P)."""
    p = np.asarray(m1, dtype=np.float64) @ np.asarray(m2, dtype=np.float64)
    p = p + _vec(bias, p.shape[0], 0.0)
    f = p.shape[0] // 2
    return gate(act, p[:f])[0] * p[f:], p


def gate_grad(dy, pre, act='silu'):
    pre, dy = np.asarray(pre, dtype=np.float64), np.asarray(dy, dtype=np.float64)
    f = pre.shape[0] // 2
    v, slope = gate(act, pre[:f])
    return np.vstack([dy * pre[f:] * slope, dy * v])


# ---- dropout

def philox4x32(counter, key, rounds=10):
    """Words (n, 4) for counters (n, 4) and one key of two words (Salmon et al., SC 2011)."""
    c = [np.asarray(counter, dtype=np.uint64)[:, j].copy() for j in range(4)]
    k = [int(key[0]), int(key[1])]
    low = np.uint64(0xFFFFFFFF)
    for _ in range(rounds):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(b >> np.uint64(32)) ^ c[1] ^ np.uint64(k[0]), b & low, (a >> np.uint64(32)) ^ c[3] ^ np.uint64(k[1]), a & low]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return np.stack(c, axis=1)


def dropout_keep(shape, dropprob, seed, stream=0, step=0.0, first=0, count=None):
    """Which entries stay, in column-major order: all of them as a matrix, or ``count`` from entry ``first`` on."""
    n = shape[0] * shape[1] if count is None else count
    g = np.arange(first // 4, (first + n + 3) // 4, dtype=np.uint64)
    bits = int(np.float32(step).view(np.uint32))
    ctr = np.stack([g & np.uint64(0xFFFFFFFF), g >> np.uint64(32), np.full_like(g, bits), np.full_like(g, stream)], axis=1)
    words = philox4x32(ctr, (seed & 0xFFFFFFFF, seed >> 32)).reshape(-1)[first % 4:][:n]
    keep = words >= np.uint64(math.floor(float(np.float32(dropprob)) * 2.0 ** 32))
    return keep if count is not None else keep.reshape(shape, order='F')


# ---- log probabilities

def is_token(labels, h):
    l = np.asarray(labels, dtype=np.float64).reshape(-1)
    with np.errstate(invalid='ignore'):
        return (l >= 0) & (l < h)


def log_probs(x, labels=None, top=0):
    """dict of logp, entropy, log_z (1 x columns) and top, top_labels (top x columns)."""
    x = np.asarray(x, dtype=np.float64)
    h, w = x.shape
    out = dict(entropy=np.empty((1, w)), log_z=np.empty((1, w)), logp=np.zeros((1, w)), top=np.empty((top, w)), top_labels=np.empty((top, w)))
    for c in range(w):
        col = x[:, c]
        ranked = np.where(np.isnan(col), -np.inf, col)
        order = np.argsort(-ranked, kind='stable')[:top]
        out['top_labels'][:, c] = order
        if np.isnan(col).any() or (col == np.inf).any():
            lp, log_z, ent = np.full(h, np.nan), np.nan, np.nan
        elif (col == -np.inf).all():
            lp, log_z, ent = np.full(h, -np.inf), -np.inf, 0.0
        else:
            m = int(np.argmax(col))
            with np.errstate(under='ignore'):
                e = np.exp(col - col[m])
            rest = float(np.sum(np.delete(e, m)))
            lz = math.log1p(rest)
            lp, log_z = (col - col[m]) - lz, col[m] + lz
            d = np.where(e > 0, col - col[m], 0.0)
            ent = lz - float(np.sum(d * e)) / (1.0 + rest)
        out['log_z'][0, c], out['entropy'][0, c] = log_z, ent
        out['top'][:, c] = lp[order]
        if labels is not None:
            l = np.asarray(labels).reshape(-1)[c]
            if is_token([l], h)[0]:
                out['logp'][0, c] = lp[int(l)]
    return out


def log_probs_grad(x, labels, log_z, logp_weight=None, entropy=None, entropy_weight=None):
    x = np.asarray(x, dtype=np.float64)
    h, w = x.shape
    row = lambda v, default: np.full((1, w), default) if v is None else np.asarray(v, dtype=np.float64).reshape(1, w)
    with np.errstate(invalid='ignore'):
        lp = x - row(log_z, 0.0)
        p = np.where(x == -np.inf, 0.0, np.exp(lp))
        spread = np.where(p == 0.0, 0.0, p * (lp + row(entropy, 0.0)))
    t = -row(entropy_weight, 0.0) * spread
    if labels is not None:
        token = is_token(labels, h).reshape(1, w)
        lw = np.where(token, row(logp_weight, 1.0), 0.0)
        t = t - lw * p
        for c in np.flatnonzero(token[0]):
            t[int(np.asarray(labels).reshape(-1)[c]), c] += lw[0, c]
    return t
