"""The operators on columns of tokens (layer norm, gated products, counter-based dropout, log probabilities of tokens) through
the C ABI against their restatements in 64 bits.

Bounds, with u = 2^-24 (half a step of fp32, relative): a sum of n terms that is taken by lanes and then over lanes is off by at most
(terms one lane adds one after the other + steps over the lanes) u times the sum of the magnitudes; `chain` below is an
upper limit for any split over at least 64 lanes (256 from 4096 terms on).  Every other operation adds u of its
result, the elementary functions a few u."""
import ctypes as ct

import numpy as np
import pytest

from oracle import token_oracle as tok

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
F = lambda a: np.asarray(a, dtype=np.float32, order='F')


def chain(n):
    return (n / 64 if n <= 4096 else n / 256) + 24


def check(got, want, bound, what=''):
    got = np.asarray(got, dtype=np.float64)
    assert got.shape == want.shape, (what, got.shape, want.shape)
    off = np.isnan(got) != np.isnan(want)
    assert not off.any(), (what, 'nan', np.argwhere(off)[:5].tolist())
    inf = np.isinf(want) | np.isinf(got)
    assert np.array_equal(got[inf], want[inf]), (what, 'inf')
    ok = ~inf & ~np.isnan(want)
    err = np.abs(got - np.where(ok, want, 0.0))
    bad = ok & ~(err <= np.broadcast_to(bound, want.shape) + 1e-44)
    assert not bad.any(), (what, np.argwhere(bad)[:5].tolist(), got[bad][:5], want[bad][:5], np.broadcast_to(bound, want.shape)[bad][:5])


def device(cm, a, skip=0):
    """The matrix on the device; with skip its columns start that many floats behind a 16-byte boundary, in the middle of others."""
    a = F(a)
    if not skip:
        return cm.CUDAMatrix(a)
    h, w = a.shape
    whole = cm.CUDAMatrix(F(np.full((h * w + skip + 5, 1), 7.25)))
    part = whole.slice(skip, skip + h * w)
    part.reshape((h, w))
    part.T = cm.TransposedCUDAMatrix(part.mat)                # (the view it had was made of the old shape)
    if a.size:
        src = cm.CUDAMatrix(a)
        part.assign(src)
        src.free_device_memory()
    part.whole = whole
    return part


def neighbours_untouched(mat, skip):
    if skip:
        v = mat.whole.asarray().ravel()
        n = mat.shape[0] * mat.shape[1]
        assert (v[:skip] == 7.25).all() and (v[skip + n:] == 7.25).all()


# ------------------------------------------------------------------ layer norm

NORM_SHAPES = [(1, 1), (1, 7), (2, 3), (3, 5), (4, 4), (10, 128), (63, 9), (64, 4), (65, 5), (100, 1), (255, 3), (256, 70), (260, 300),
               (1000, 33), (1001, 17), (1024, 4), (2046, 11), (2048, 300), (2050, 5), (4096, 9), (4099, 3), (8192, 5), (8196, 3),
               (10000, 2), (16384, 2), (16390, 3), (20000, 3), (40001, 2), (70000, 1), (12, 5000), (7, 3001)]


def norm_inputs(rng, h, w):
    x = rng.standard_normal((h, w)) * np.exp(rng.standard_normal((1, w))) + rng.standard_normal((1, w))
    return F(x), F(1 + 0.3 * rng.standard_normal((h, 1))), F(rng.standard_normal((h, 1)))


def norm_bound(x, gain, y):
    """The normalised value is (x - mean) * r: the mean is off by chain u of the mean deviation, r by chain u."""
    h = x.shape[0]
    xh, _ = tok.normalised(x, 1e-5)
    g = 1.0 if gain is None else np.abs(gain.astype(np.float64))
    return U * (g * (np.abs(xh) * (chain(h) + 8) + chain(h) * np.abs(xh).mean(axis=0, keepdims=True)) + 2 * np.abs(y))


@pytest.mark.parametrize("h,w", NORM_SHAPES)
@pytest.mark.parametrize("skip", [0, 1])
def test_layer_norm(cm, rng, h, w, skip):
    x, gain, bias = norm_inputs(rng, h, w)
    for g, b in ((gain, bias), (gain, None), (None, bias), (None, None)):
        y = device(cm, np.zeros((h, w)), skip)
        cm.layer_norm(device(cm, x, skip), None if g is None else cm.CUDAMatrix(g), None if b is None else cm.CUDAMatrix(b), target=y)
        want = tok.layer_norm(x, g, b)
        check(y.asarray(), want, norm_bound(x, g, want), (h, w, skip))
        neighbours_untouched(y, skip)
    m = device(cm, x, skip)
    assert cm.layer_norm(m, cm.CUDAMatrix(gain), cm.CUDAMatrix(bias)) is m           # in place
    want = tok.layer_norm(x, gain, bias)
    check(m.asarray(), want, norm_bound(x, gain, want), 'in place')
    neighbours_untouched(m, skip)


@pytest.mark.parametrize("h", [5, 64, 1000, 5000, 40000])
def test_layer_norm_far_from_zero_and_special_columns(cm, rng, h):
    """A mean 10^4 deviations from zero costs no digits of the deviations (x is exact, so the oracle sees the same numbers); a
    constant column gives the bias; a column with NaN or infinity is NaN, its neighbours are not."""
    x = rng.standard_normal((h, 8))
    x[:, 1] += 1e4
    x[:, 2] = 3.0
    x[:, 3] = -1e-3 + 1e-9 * x[:, 3]
    x = F(x)
    x[h // 2, 4], x[0, 5], x[h - 1, 6] = np.nan, np.inf, -np.inf
    bias = F(rng.standard_normal((h, 1)))
    got = cm.layer_norm(cm.CUDAMatrix(x), bias=cm.CUDAMatrix(bias), target=cm.empty(x.shape)).asarray()
    ok = [0, 1, 2, 3, 7]
    want = tok.layer_norm(x[:, ok], None, bias)
    check(got[:, ok], want, norm_bound(x[:, ok], None, want))
    assert np.array_equal(got[:, 2], bias[:, 0])
    assert np.isnan(got[:, 4:7]).all()


def grad_bounds(dy, x, gain):
    h, w = x.shape
    xh, r = tok.normalised(x, 1e-5)
    xa, dya = np.abs(xh), np.abs(dy.astype(np.float64))
    g = dya * (1.0 if gain is None else np.abs(gain.astype(np.float64)))
    k = chain(h) + 8
    ma, mb = g.mean(axis=0, keepdims=True), (g * (xa + 1)).mean(axis=0, keepdims=True)
    # x^ is off by k u (|x^| + 1); every product and mean by k u of its magnitudes
    dx = U * r * (k + 4) * (g + ma + 3 * (xa + 1) * mb)
    rows = w / 4 + 24 + k
    return dx, U * rows * (dya * (xa + 1)).sum(axis=1, keepdims=True), U * (w / 4 + 24) * dya.sum(axis=1, keepdims=True)


@pytest.mark.parametrize("h,w", NORM_SHAPES + [(64, 127), (33, 128), (64, 129), (256, 31), (200, 32), (200, 33), (1024, 8), (1024, 9), (700, 5), (1, 70000), (2, 400), (3, 200001), (4, 30001), (1000, 700), (516, 2049), (4098, 130)])
@pytest.mark.parametrize("skip", [0, 1])
def test_layer_norm_grad(cm, rng, h, w, skip):
    x, gain, _ = norm_inputs(rng, h, w)
    dy = F(rng.standard_normal((h, w)) + 0.2)
    for g in (gain, None):
        G = None if g is None else cm.CUDAMatrix(g)
        dx, gg, bg = device(cm, np.zeros((h, w)), skip), cm.empty((h, 1)), cm.empty((h, 1))
        gg.assign(np.nan); bg.assign(np.nan)                        # beta = 0 reads nothing
        cm.layer_norm_grad(device(cm, dy, skip), device(cm, x, skip), G, target=dx, gain_grad=gg, bias_grad=bg)
        want = tok.layer_norm_grad(dy, x, g)
        for got, wt, bd, what in zip((dx, gg, bg), want, grad_bounds(dy, x, g), ('dx', 'gain', 'bias')):
            check(got.asarray(), wt, bd + U * np.abs(wt), (what, h, w, skip))
        neighbours_untouched(dx, skip)
    # accumulated, and in the place of either input; one of the parameters alone, or none
    wt, bd = tok.layer_norm_grad(dy, x, gain), grad_bounds(dy, x, gain)
    old = F(rng.standard_normal((h, 2)))
    gg, bg = cm.CUDAMatrix(old[:, :1]), cm.CUDAMatrix(old[:, 1:])
    d = device(cm, dy, skip)
    assert cm.layer_norm_grad(d, device(cm, x, skip), cm.CUDAMatrix(gain), gain_grad=gg, mult=0.25, beta=1.0) is d
    check(d.asarray(), wt[0], bd[0] + U * np.abs(wt[0]), 'in place of deriv')
    check(gg.asarray(), old[:, :1] + 0.25 * wt[1], 0.25 * bd[1] + 3 * U * (np.abs(old[:, :1]) + np.abs(wt[1])), 'added')
    m = device(cm, x, skip)
    cm.layer_norm_grad(device(cm, dy, skip), m, cm.CUDAMatrix(gain), target=m, bias_grad=bg, mult=-2.0, beta=0.5)
    check(m.asarray(), wt[0], bd[0] + U * np.abs(wt[0]), 'in place of mat')
    check(bg.asarray(), 0.5 * old[:, 1:] - 2.0 * wt[2], 2 * bd[2] + 3 * U * (np.abs(old[:, 1:]) + 2 * np.abs(wt[2])), 'scaled')
    d = device(cm, dy, skip)
    cm.layer_norm_grad(d, device(cm, x, skip), cm.CUDAMatrix(gain))
    check(d.asarray(), wt[0], bd[0] + U * np.abs(wt[0]), 'inputs alone')


@pytest.mark.parametrize("h,w", [(1026, 3000), (2049, 3000), (4097, 1500), (9001, 600)])
def test_layer_norm_and_its_gradient_give_the_same_bits_every_time(cm, rng, h, w):
    """Heights whose last group of four rows overlaps one that a lane of another wavefront has."""
    x, gain, bias = (cm.CUDAMatrix(v) for v in norm_inputs(rng, h, w))
    dy = cm.CUDAMatrix(F(rng.standard_normal((h, w))))
    def run():
        y, dx, gg, bg = cm.empty((h, w)), cm.empty((h, w)), cm.empty((h, 1)), cm.empty((h, 1))
        cm.layer_norm(x, gain, bias, target=y)
        cm.layer_norm_grad(dy, x, gain, target=dx, gain_grad=gg, bias_grad=bg)
        return [m.asarray().tobytes() for m in (y, dx, gg, bg)]
    first = run()
    assert all(run() == first for _ in range(5))


def test_layer_norm_of_no_columns_or_rows(cm):
    none, v = cm.empty((5, 0)), cm.CUDAMatrix(F(np.ones((5, 1))))
    cm.layer_norm(none, v, v, target=cm.empty((5, 0)))
    gg, bg = cm.CUDAMatrix(F(np.full((5, 1), 3.0))), cm.CUDAMatrix(F(np.full((5, 1), np.nan)))
    cm.layer_norm_grad(cm.empty((5, 0)), none, v, target=cm.empty((5, 0)), gain_grad=gg, beta=2.0)
    cm.layer_norm_grad(cm.empty((5, 0)), none, v, target=cm.empty((5, 0)), bias_grad=bg)
    assert (gg.asarray() == 6.0).all() and (bg.asarray() == 0.0).all()             # sums of nothing
    cm.layer_norm(cm.empty((0, 4)), target=cm.empty((0, 4)))
    cm.layer_norm_grad(cm.empty((0, 4)), cm.empty((0, 4)))


# ------------------------------------------------------------------ gated products

ACTS = [None, 'sigmoid', 'relu', 'tanh', 'silu', 'gelu']


def act_bounds(act, p, perr):
    """How far act(gate) and its slope may be off where the gate is off by perr: the slopes are at most 1.2 and the curvatures 1
    in magnitude; the functions themselves 16 u, and gelu's share of the normal distribution 2 gate^2 u more (its argument's rounding)."""
    v, s = tok.gate(act, p)
    rel = 16 + (2 * np.minimum(p * p, 250.0) if act == 'gelu' else 0)
    flip = (np.abs(p) <= perr) if act == 'relu' else 0.0
    return 1.2 * perr + U * rel * np.abs(v), perr + U * (rel * np.abs(s) + 8 * np.abs(v) + 8) + flip


def gated_check(cm, w, x, bias, act, got, pre):
    want, p = tok.dot_gated(w.T, x, bias, act)
    k = w.shape[0]
    perr = U * ((k / 4 + 24) * (np.abs(w.T.astype(np.float64)) @ np.abs(x.astype(np.float64))) + 2 * np.abs(p))
    if bias is not None:
        perr = perr + U * np.abs(bias)
    f = p.shape[0] // 2
    v, _ = tok.gate(act, p[:f])
    verr, _ = act_bounds(act, p[:f], perr[:f])
    check(got, want, verr * (np.abs(p[f:]) + perr[f:]) + np.abs(v) * perr[f:] + 4 * U * np.abs(want), ('gated', w.shape, x.shape, act))
    if pre is not None:
        check(pre, p, perr, 'pre')


# inputs, units, columns
GATED_SHAPES = [(1, 1, 1), (1, 3, 2), (3, 1, 5), (5, 7, 1), (64, 64, 1), (65, 63, 2), (100, 33, 3), (128, 40, 4), (127, 129, 7), (300, 250, 8),
                (500, 1000, 9), (256, 64, 16), (1001, 517, 1), (1000, 130, 17), (64, 512, 64), (333, 301, 65), (1024, 640, 33),
                (200, 700, 300), (2048, 300, 5), (300, 700, 9), (1001, 33, 13), (260, 5000, 15), (129, 16, 11), (2049, 128, 2), (4100, 70, 1), (64, 128, 128), (40, 256, 384), (256, 1024, 512),
                (1001, 1500, 300), (520, 1030, 777), (31, 2048, 1024), (512, 2050, 1030), (32, 32, 64), (33, 35, 67), (63, 100, 500), (70, 300, 40),
                (64, 1000, 33), (130, 40, 31), (128, 17, 20), (1001, 257, 65), (71, 160, 10), (40, 33, 9),
                (127, 64, 31), (5, 7, 13), (100, 1000, 20), (97, 2100, 25), (3, 2, 32)]


@pytest.mark.parametrize("d,f,n", GATED_SHAPES)
def test_dot_gated(cm, rng, d, f, n):
    w, x, bias = F(rng.standard_normal((d, 2 * f)) / np.sqrt(d)), F(rng.standard_normal((d, n))), F(0.3 * rng.standard_normal((2 * f, 1)))
    W, X, B = cm.CUDAMatrix(w), cm.CUDAMatrix(x), cm.CUDAMatrix(bias)
    for act, b, keep in (('silu', False, False), ('gelu', True, True), ('relu', False, True), ('sigmoid', True, False), ('tanh', False, False), (None, True, True)):
        y, pre = device(cm, np.zeros((f, n)), 1 if act == 'gelu' else 0), cm.empty((2 * f, n)) if keep else None
        cm.dot_gated(W.T, X, B if b else None, target=y, act=act, pre=pre)
        gated_check(cm, w, x, bias if b else None, act, y.asarray(), pre.asarray() if keep else None)
        if act == 'gelu':
            neighbours_untouched(y, 1)
    assert cm.dot_gated(W.T, X).shape == (f, n)


@pytest.mark.parametrize("d,f,n", [(5, 7, 1), (65, 63, 2), (300, 250, 8), (1001, 517, 3), (333, 301, 65), (64, 128, 128), (520, 1030, 777), (260, 1028, 512)])
@pytest.mark.parametrize("stored", ["nn", "nt", "tt"])
@pytest.mark.parametrize("skip", [0, 1])
def test_dot_gated_of_operands_stored_either_way(cm, rng, d, f, n, stored, skip):
    w, x = F(rng.standard_normal((d, 2 * f)) / np.sqrt(d)), F(rng.standard_normal((d, n)))
    W = device(cm, w.T, skip) if stored[0] == 'n' else device(cm, w, skip).T
    X = device(cm, x, skip) if stored[1] == 'n' else device(cm, x.T, skip)
    y, pre = cm.empty((f, n)), cm.empty((2 * f, n))
    cm.dot_gated(W, X if stored[1] == 'n' else X.T, target=y, pre=pre)
    gated_check(cm, w, x, None, 'silu', y.asarray(), pre.asarray())


def test_dot_gated_takes_infinities_and_nan_where_they_are(cm, rng):
    """One column of the inputs with NaN, one with infinity: theirs are the results that are not finite."""
    for d, f, n in ((64, 40, 6), (300, 700, 300), (1024, 1500, 1500), (64, 40, 11), (2048, 30, 6)):
        w, x = F(rng.standard_normal((d, 2 * f)) / np.sqrt(d)), F(rng.standard_normal((d, n)))
        x[3, 1], x[5, 4] = np.nan, np.inf
        y = cm.dot_gated(cm.CUDAMatrix(w).T, cm.CUDAMatrix(x), act='sigmoid').asarray()
        ok = [c for c in range(n) if c not in (1, 4)]
        gated_check(cm, w, x[:, ok], None, 'sigmoid', y[:, ok], None)
        assert np.isnan(y[:, 1]).all() and not np.isfinite(y[:, 4]).all()


def test_gates_far_from_zero(cm):
    """Products of one term, exact: the activations over the whole range, with the limits behind it."""
    g = np.concatenate([np.linspace(-100, 100, 4001), [0.0, -0.0, 1e-30, -1e-30, 1e4, -1e4, -13.0, -14.5]])
    w = F(np.concatenate([g, np.ones_like(g)]).reshape(1, -1))
    one = F(np.ones((1, 1)))
    g = w[0, :g.size].astype(np.float64)
    for act in ACTS:
        pre = cm.empty((w.shape[1], 1))
        y = cm.dot_gated(cm.CUDAMatrix(w).T, cm.CUDAMatrix(one), act=act, pre=pre).asarray()
        v, s = tok.gate(act, g.reshape(-1, 1))
        ve, se = act_bounds(act, g.reshape(-1, 1), 0.0)
        check(y, v, ve + 1e-38, act)
        d = cm.dot_gated_grad(cm.CUDAMatrix(F(np.ones_like(y))), cm.CUDAMatrix(w).T, cm.CUDAMatrix(one), pre, act=act).asarray()
        check(d, np.vstack([s, v]), np.vstack([se, ve + 1e-38]), act)


@pytest.mark.parametrize("d,f,n", [(1, 1, 1), (5, 7, 1), (65, 63, 2), (258, 300, 1), (1027, 70, 3), (2048, 2500, 4), (300, 33, 5), (513, 64, 6), (64, 1000, 7), (1000, 517, 8), (100, 33, 30), (127, 129, 64), (500, 1000, 100), (333, 301, 257), (64, 520, 512), (256, 1024, 1024)])
@pytest.mark.parametrize("act", ACTS)
def test_dot_gated_grad(cm, rng, d, f, n, act):
    w, x, dy = F(rng.standard_normal((d, 2 * f)) / np.sqrt(d)), F(rng.standard_normal((d, n))), F(rng.standard_normal((f, n)))
    pre = F(1.5 * rng.standard_normal((2 * f, n)))
    W, X, PRE, DY = cm.CUDAMatrix(w), cm.CUDAMatrix(x), cm.CUDAMatrix(pre), cm.CUDAMatrix(dy)
    t, dw, dx, db = cm.empty((2 * f, n)), cm.empty((d, 2 * f)), cm.empty((d, n)), cm.empty((2 * f, 1))
    for m in (dw, dx, db):
        m.assign(np.nan)
    assert cm.dot_gated_grad(DY, W.T, X, PRE, target=t, m1_grad=dw, m2_grad=dx, bias_grad=db, act=act) is t
    want = tok.gate_grad(dy, pre, act)
    ve, se = act_bounds(act, pre[:f].astype(np.float64), 0.0)
    ad, au = np.abs(dy.astype(np.float64)), np.abs(pre[f:].astype(np.float64))
    terr = np.vstack([ad * au * se, ad * ve]) + 4 * U * np.abs(want)
    check(t.asarray(), want, terr, ('halves', act))
    aw, ax, at = np.abs(w.astype(np.float64)), np.abs(x.astype(np.float64)), np.abs(want)
    wdw, wdx, wdb = x.astype(np.float64) @ want.T, w.astype(np.float64) @ want, want.sum(axis=1, keepdims=True)
    edw = ax @ terr.T + U * (n / 4 + 24) * (ax @ at.T)
    edx = aw @ terr + U * (f / 2 + 24) * (aw @ at)
    edb = terr.sum(axis=1, keepdims=True) + U * (n / 4 + 24) * at.sum(axis=1, keepdims=True)
    check(dw.asarray(), wdw, edw, 'weights'); check(dx.asarray(), wdx, edx, 'inputs'); check(db.asarray(), wdb, edb, 'bias')
    # accumulated; in the place of pre; one gradient alone
    old = F(rng.standard_normal((d, 2 * f)))
    dw, db = cm.CUDAMatrix(old), cm.CUDAMatrix(F(np.full((2 * f, 1), 2.0)))
    assert cm.dot_gated_grad(DY, W.T, X, PRE, m1_grad=dw, bias_grad=db, act=act, mult=0.5, beta=1.0) is PRE
    assert np.array_equal(PRE.asarray(), t.asarray())
    check(dw.asarray(), old + 0.5 * wdw, 0.5 * edw + 3 * U * (np.abs(old) + np.abs(wdw)), 'added')
    check(db.asarray(), 2.0 + 0.5 * wdb, 0.5 * edb + 3 * U * (2 + np.abs(wdb)), 'added')
    PRE = cm.CUDAMatrix(pre)
    db = cm.CUDAMatrix(F(np.full((2 * f, 1), 2.0)))
    cm.dot_gated_grad(DY, W.T, X, PRE, target=t, bias_grad=db, act=act, mult=-2.0, beta=0.25)
    check(db.asarray(), 0.5 - 2.0 * wdb, 2 * edb + 3 * U * (1 + 2 * np.abs(wdb)), 'scaled')


@pytest.mark.parametrize("d,f,n", [(4, 3, 1), (5, 30, 8), (258, 130, 3), (1030, 700, 8), (2051, 100, 1), (300, 64, 64), (3, 9, 2), (7, 20, 9), (300, 260, 13), (1027, 130, 16)])
def test_dot_gated_grad_of_one_operand_alone_and_accumulated(cm, rng, d, f, n):
    """Which gradients are asked for does not change them; all of them accumulated."""
    w, x, dy = F(rng.standard_normal((d, 2 * f)) / np.sqrt(d)), F(rng.standard_normal((d, n))), F(rng.standard_normal((f, n)))
    W, X, PRE, DY = cm.CUDAMatrix(w), cm.CUDAMatrix(x), cm.CUDAMatrix(F(rng.standard_normal((2 * f, n)))), cm.CUDAMatrix(dy)
    def run(names, old=np.nan, **scales):
        t, out = cm.empty((2 * f, n)), dict(m1_grad=(d, 2 * f), m2_grad=(d, n), bias_grad=(2 * f, 1))
        out = {k: cm.CUDAMatrix(F(np.full(out[k], old))) for k in names}
        cm.dot_gated_grad(DY, W.T, X, PRE, target=t, **out, **scales)
        return t.asarray().astype(np.float64), {k: m.asarray().copy() for k, m in out.items()}
    t, every = run(('m1_grad', 'm2_grad', 'bias_grad'))
    at, chains = np.abs(t), U * (n / 4 + 24)
    edw, edb = chains * (np.abs(x.astype(np.float64)) @ at.T), chains * at.sum(axis=1, keepdims=True)
    edx = U * (f / 2 + 24) * (np.abs(w.astype(np.float64)) @ at)
    wdw, wdx, wdb = x.astype(np.float64) @ t.T, w.astype(np.float64) @ t, t.sum(axis=1, keepdims=True)
    for names in (('m1_grad',), ('m2_grad',), ('bias_grad',), ('m1_grad', 'm2_grad'), ('m2_grad', 'bias_grad'), tuple(every)):
        _, got = run(names)
        for k, want, bound in (('m1_grad', wdw, edw), ('m2_grad', wdx, edx), ('bias_grad', wdb, edb)):
            if k in names:
                check(got[k], want, bound, (names, k))
    _, got = run(tuple(every), old=3.0, beta=0.5, mult=-2.0)
    check(got['m1_grad'], 1.5 - 2 * wdw, 2 * edw + 3 * U * (1.5 + 2 * np.abs(wdw)), 'added')
    check(got['m2_grad'], wdx, edx, 'not added')
    check(got['bias_grad'], 1.5 - 2 * wdb, 2 * edb + 3 * U * (1.5 + 2 * np.abs(wdb)), 'added')


def test_dot_gated_grad_of_operands_stored_either_way(cm, rng):
    d, f, n = 70, 33, 20
    w, x, dy = F(rng.standard_normal((d, 2 * f))), F(rng.standard_normal((d, n))), F(rng.standard_normal((f, n)))
    pre = F(rng.standard_normal((2 * f, n)))
    t = tok.gate_grad(dy, pre, 'silu')
    wdw, wdx = x.astype(np.float64) @ t.T, w.astype(np.float64) @ t
    edw = U * 64 * (np.abs(x.astype(np.float64)) @ np.abs(t.T) + 1); edx = U * 64 * (np.abs(w.astype(np.float64)) @ np.abs(t) + 1)
    for wt in (False, True):
        for xt in (False, True):
            W, X = cm.CUDAMatrix(F(w if wt else w.T)), cm.CUDAMatrix(F(x.T if xt else x))
            dw, dx = cm.empty(W.shape), cm.empty(X.shape)
            cm.dot_gated_grad(cm.CUDAMatrix(dy), W.T if wt else W, X.T if xt else X, cm.CUDAMatrix(pre), m1_grad=dw, m2_grad=dx)
            check(dw.asarray() if wt else dw.asarray().T, wdw, edw, (wt, xt))
            check(dx.asarray().T if xt else dx.asarray(), wdx, edx, (wt, xt))


def test_gated_of_no_columns(cm):
    w = cm.CUDAMatrix(F(np.ones((3, 8))))
    cm.dot_gated(w.T, cm.empty((3, 0)), target=cm.empty((4, 0)))
    dw, db = cm.CUDAMatrix(F(np.full((3, 8), 2.0))), cm.CUDAMatrix(F(np.full((8, 1), np.nan)))
    cm.dot_gated_grad(cm.empty((4, 0)), w.T, cm.empty((3, 0)), cm.empty((8, 0)), m1_grad=dw, beta=0.5)
    cm.dot_gated_grad(cm.empty((4, 0)), w.T, cm.empty((3, 0)), cm.empty((8, 0)), bias_grad=db)
    assert (dw.asarray() == 1.0).all() and (db.asarray() == 0.0).all()
    y = cm.dot_gated(cm.empty((0, 8)).T, cm.empty((0, 5)), bias=cm.CUDAMatrix(F(np.full((8, 1), 2.0))), act='relu')       # no terms
    assert (y.asarray() == 4.0).all()


# ------------------------------------------------------------------ dropout

@pytest.mark.parametrize("h,w", [(1, 1), (1, 3), (3, 3), (4, 1), (5, 5), (10, 128), (1001, 33), (1024, 100), (4096, 257), (13, 5000)])
@pytest.mark.parametrize("skip", [0, 1])
def test_counter_dropout(cm, rng, h, w, skip):
    x, r = F(rng.standard_normal((h, w))), F(rng.standard_normal((h, w)))
    step = cm.CUDAMatrix(F([[41.0]]))
    seed, stream = 0xfedcba9876543210, 0xfffffffe
    for p in (0.0, 0.1, 0.5, 0.9375, 1.0):
        mult = np.float32(1.0 / (1.0 - p) if p < 1 else 0.0)
        keep = tok.dropout_keep((h, w), p, seed, stream, 41.0)
        y = device(cm, np.zeros((h, w)), skip)
        cm.counter_dropout(device(cm, x, skip), p, seed, stream=stream, step=step, target=y)
        assert np.array_equal(y.asarray(), np.where(keep, x * mult, np.float32(0))), p
        neighbours_untouched(y, skip)
        y = device(cm, x, skip)
        cm.counter_dropout(y, p, seed, stream=stream, step=step, mult=1.5, residual=device(cm, r, skip))       # in place, one rounding
        want = r.astype(np.float64) + np.where(keep, x.astype(np.float64) * 1.5, 0.0)
        check(y.asarray(), want, U * np.abs(want), p)
        t = device(cm, r, skip)
        cm.counter_dropout(device(cm, x, skip), p, seed, stream=stream, step=step, mult=1.5, residual=t, target=t)
        assert np.array_equal(t.asarray(), y.asarray())
    y = cm.counter_dropout(device(cm, x, skip), 0.5, seed, mult=-np.inf, residual=device(cm, r, skip)).asarray()       # any factor
    keep = tok.dropout_keep((h, w), 0.5, seed)
    assert np.array_equal(y[~keep], r[~keep]) and not np.isfinite(y[keep]).any()
    keep = tok.dropout_keep((h, w), 0.5, 7)                 # no step, first stream; what is dropped may be anything
    x[~keep] = [np.nan, np.inf, -np.inf][h % 3]
    y = cm.counter_dropout(device(cm, x, skip), 0.5, 7, mult=1.0).asarray()
    assert np.array_equal(y, np.where(keep, x, np.float32(0))) and not np.signbit(y[~keep]).any()


def test_counter_dropout_depends_on_seed_stream_and_step(cm):
    x = cm.CUDAMatrix(F(np.ones((100, 100))))
    def mask(seed, stream=0, step=None):
        s = None if step is None else cm.CUDAMatrix(F([[step]]))
        return cm.counter_dropout(x, 0.5, seed, stream=stream, step=s, mult=1.0, target=cm.empty((100, 100))).asarray()
    base = mask(5)
    assert np.array_equal(base, mask(5, step=0.0)) and np.array_equal(base, mask(5))
    for other in (mask(6), mask(5 + (1 << 32)), mask(5, 1), mask(5, 0, 1.0)):
        assert 0.4 < np.mean(other == base) < 0.6


# ------------------------------------------------------------------ log probabilities

LOGP_SHAPES = [(1, 1), (1, 5), (2, 3), (3, 300), (10, 128), (63, 5), (64, 3), (65, 7), (100, 40), (257, 9), (1000, 33), (1001, 5), (1024, 64), (2050, 3), (1500, 2100),
               (2050, 2048), (3074, 2049), (4096, 17), (4099, 2), (8192, 3), (10007, 5), (16384, 40), (32003, 4), (50000, 1), (50001, 2), (128256, 1), (131072, 3), (300007, 1)]


def logp_bounds(x, labels, o):
    """r, the sum of e^d over the others than the maximum m, is off by (chain + 8) u: of log(1 + r) that is r / (1 + r) as much.
    d = x - m is itself rounded, by u |d| at most, which makes e^(d + u d) = e^d (1 + u d): r is off by u sum |d| e^d more, and
    sum |d| e^d / (1 + r) is entropy - log(1 + r).  The entropy's own sum of d e^d is off by u d^2 e^d a term in the same way,
    and |d| is at most 104 where e^d is not 0 in fp32."""
    h = x.shape[0]
    with np.errstate(invalid='ignore', divide='ignore'):
        lz = o['log_z'] - np.max(np.where(np.isnan(x), -np.inf, x).astype(np.float64), axis=0, keepdims=True)
        share = -np.expm1(-lz)
        k = U * ((chain(h) + 8) * share + np.abs(o['entropy'] - lz))
        spread = np.abs(o['entropy']) + lz
        b = dict(log_z=U * np.abs(o['log_z']) + k, logp=2 * U * np.abs(o['logp']) + k, top=2 * U * np.abs(o['top']) + k)
        b['entropy'] = 2 * U * np.abs(o['entropy']) + k + U * (2 * chain(h) + 16 + 105) * (np.abs(spread) + share)
    return {n: np.where(np.isfinite(v), v, 0.0) for n, v in b.items()}


def run_log_probs(cm, x, labels, k, skip=0, **without):
    h, w = x.shape
    out = {n: device(cm, np.full((1, w), 9.0), skip) for n in ('logp', 'entropy', 'log_z')}
    if k:
        out.update(top=device(cm, np.full((k, w), 9.0), skip), top_labels=device(cm, np.full((k, w), 9.0), skip))
    cm.log_probs(device(cm, x, skip), cm.CUDAMatrix(labels), **out)
    got = {n: m.asarray().copy() for n, m in out.items()}
    for m in out.values():
        neighbours_untouched(m, skip)
    return got


def check_log_probs(x, labels, k, got):
    o = tok.log_probs(x, labels, k)
    b = logp_bounds(x, labels, o)
    for n in got:
        if n == 'top_labels':
            assert np.array_equal(got[n], o[n]), (x.shape, k, np.argwhere(got[n] != o[n])[:5].tolist())
        else:
            check(got[n], o[n], b[n], (n, x.shape, k))
    return o


@pytest.mark.parametrize("h,w", LOGP_SHAPES)
@pytest.mark.parametrize("skip", [0, 1])
def test_log_probs(cm, rng, h, w, skip):
    x = F(3 * rng.standard_normal((h, w)))
    labels = F(rng.integers(-1, h + 1, (1, w)))
    for k in sorted({0, 1, min(h, 5), min(h, 20), min(h, 64)}):
        check_log_probs(x, labels, k, run_log_probs(cm, x, labels, k, skip))


@pytest.mark.parametrize("h", [5, 64, 100, 1000, 5000, 40000, 200000])
def test_log_probs_of_ties_masks_and_special_columns(cm, rng, h):
    w, lowest = 16, np.finfo(np.float32).min
    x = F(rng.standard_normal((h, w)))
    x[:, 0] = 0.25                                             # all alike
    x[:, 1] = -np.inf                                          # a mask that leaves nothing
    x[:, 2] = lowest                                           # ... of the type's lowest value
    x[1:, 3] = -np.inf                                         # one entry left, the first
    x[:-1, 4] = lowest                                         # ... the last
    x[:, 5] = np.round(x[:, 5])                                # many ties
    x[::2, 6] = -np.inf
    x[h // 2, 7] = np.nan
    x[:, 8] = np.nan
    x[h - 1, 9] = np.inf
    x[0, 10], x[h - 1, 10] = 60.0, 60.0                        # two that have nearly everything
    x[h // 3, 11] = 40.0                                       # one that has: log p of -1e-13 or so
    x[:, 12] *= 1e30
    x[:, 13] = np.sort(x[:, 13])                               # the best ones last
    x[:, 14] = np.sort(x[:, 14])[::-1]                         # ... first
    x[:, 15] = np.where(np.arange(h) % 2, 0.0, -0.0)           # equal zeros
    labels = F(rng.integers(0, h, (1, w)))
    labels[0, [3, 4, 10, 11]] = 0, h - 1, 0, h // 3
    labels[0, 13], labels[0, 14] = np.nan, -0.5                # no tokens
    for k in sorted({min(h, 5), min(h, 64)}):
        o = check_log_probs(x, labels, k, run_log_probs(cm, x, labels, k))
    assert o['logp'][0, 1] == -np.inf and o['logp'][0, 13] == 0 and o['logp'][0, 14] == 0 and (h < 100 or -1e-10 < o['logp'][0, 11] < 0)


@pytest.mark.parametrize("h,w", [(40000, 600), (131072, 2), (60001, 700)])
def test_log_probs_where_the_best_entries_are_close_together(cm, rng, h, w):
    """Groups of four rows at a distance of 256 groups go to the same lane of a workgroup: with the large entries in a few lanes, far more
    entries than asked for are candidates; with them in one run of rows, every lane has some."""
    x = F(rng.standard_normal((h, w)))
    rows = np.arange(h)
    for c in range(w):
        if c % 3 == 0:
            x[(rows // 4) % 256 < 19, c] += 100.0
        elif c % 3 == 1:
            x[h // 2:h // 2 + 3000, c] += 50.0
    labels = F(rng.integers(0, h, (1, w)))
    X = cm.CUDAMatrix(x)
    t, l = cm.empty((20, w)), cm.empty((20, w))
    cm.log_probs(X, top=t, top_labels=l)
    got, probs = l.asarray(), t.asarray()
    for c in list(range(min(w, 9))) + [w - 1]:
        order = np.argsort(-x[:, c].astype(np.float64), kind='stable')[:20]
        assert np.array_equal(got[:, c], order), c
    o = tok.log_probs(x[:, :4], labels[:, :4], 20)
    check(probs[:, :4], o['top'][:, :w], logp_bounds(x[:, :4], labels[:, :4], o)['top'], 'top')


def test_log_probs_gives_what_is_asked_for(cm, rng):
    x, labels = F(rng.standard_normal((300, 6))), F(rng.integers(0, 300, (1, 6)))
    X, L = cm.CUDAMatrix(x), cm.CUDAMatrix(labels)
    o = tok.log_probs(x, labels, 4)
    assert np.allclose(cm.log_probs(X, L).asarray(), o['logp'], rtol=1e-5)
    e, t, l = cm.empty((1, 6)), cm.empty((4, 6)), cm.empty((4, 6))
    assert cm.log_probs(X, entropy=e) is None and np.allclose(e.asarray(), o['entropy'], rtol=1e-5)
    cm.log_probs(X, top=t); cm.log_probs(X, top_labels=l)
    assert np.allclose(t.asarray(), o['top'], rtol=1e-5) and np.array_equal(l.asarray(), o['top_labels'])
    cm.log_probs(cm.empty((300, 0)), entropy=cm.empty((1, 0)))
    z, e, p = (cm.CUDAMatrix(F(np.full((1, 3), 9.0))) for _ in range(3))                  # no rows: no distribution
    cm.log_probs(cm.empty((0, 3)), cm.CUDAMatrix(F(np.zeros((1, 3)))), p, e, z)
    assert (z.asarray() == -np.inf).all() and (e.asarray() == 0).all() and (p.asarray() == 0).all()
    cm.log_probs_grad(cm.empty((0, 3)), None, z)


@pytest.mark.parametrize("h,w", LOGP_SHAPES)
@pytest.mark.parametrize("skip", [0, 1])
def test_log_probs_grad(cm, rng, h, w, skip):
    x, labels = F(3 * rng.standard_normal((h, w))), F(rng.integers(-1, h + 1, (1, w)))
    lw, ew = F(rng.standard_normal((1, w))), F(rng.standard_normal((1, w)))
    if w > 2:
        x[h // 2:, 1] = -np.inf
        x[:, 2] = -np.inf
    o = tok.log_probs(x, labels)
    z, ent = F(o['log_z']), F(o['entropy'])
    D = cm.CUDAMatrix
    for l, a, e in ((labels, lw, ew), (labels, lw, None), (labels, None, None), (None, None, ew)):
        t = device(cm, np.full((h, w), 5.0), skip)
        cm.log_probs_grad(device(cm, x, skip), None if l is None else D(l), D(z), None if a is None else D(a), None if e is None else D(ent),
                          None if e is None else D(e), target=t)
        want = tok.log_probs_grad(x, l, z, a, None if e is None else ent, e)
        # log p is off by u of itself, p by (|log p| + 8) u, p (log p + entropy) by that much more
        with np.errstate(invalid='ignore'):
            lp = np.where(np.isfinite(x - z.astype(np.float64)), x - z.astype(np.float64), 0.0)
        p = np.where(np.isfinite(x), np.exp(lp), 0.0)
        al = np.abs(lp) + 8
        aw = 0.0 if l is None else np.abs(lw if a is not None else 1.0)
        ae = 0.0 if e is None else np.abs(ew.astype(np.float64))
        bound = U * (p * al * (2 * aw + ae * (2 * np.abs(lp) + 2 * np.abs(ent) + 2)) + 4 * np.abs(want))
        check(t.asarray(), want, bound + 1e-38, (h, w, skip))
        neighbours_untouched(t, skip)
    m = device(cm, x, skip)
    assert cm.log_probs_grad(m, D(labels), D(z), D(lw), D(ent), D(ew)) is m                     # in place
    t = cm.empty((h, w))
    cm.log_probs_grad(D(x), D(labels), D(z), D(lw), D(ent), D(ew), target=t)
    assert np.array_equal(m.asarray(), t.asarray())


def test_log_probs_grad_is_the_classifier_loss_gradient(cm, rng):
    """With weights of -1: the gradient that softmax_ce_grad gives."""
    x, labels = F(rng.standard_normal((50, 30))), F(rng.integers(0, 50, (1, 30)))
    X, L = cm.CUDAMatrix(x), cm.CUDAMatrix(labels)
    z, minus = cm.empty((1, 30)), cm.CUDAMatrix(F(np.full((1, 30), -1.0)))
    cm.log_probs(X, L, log_z=z)
    got = cm.log_probs_grad(X, L, z, minus, target=cm.empty((50, 30))).asarray()
    grad = cm.empty((50, 30))
    cm.softmax_ce_grad(X, L, probs=cm.empty((50, 30)), grad=grad)
    assert np.max(np.abs(got - grad.asarray())) < 1e-6


# ------------------------------------------------------------------ together

class Block(object):
    """A feed-forward block over tokens with its loss: x + dropout(w2^T gated(norm(x))), norm, logits, log probabilities; and back."""

    def __init__(self, cm, rng, d=96, f=160, v=1000, n=70):
        self.cm, self.shape = cm, (d, f, v, n)
        D = lambda a: cm.CUDAMatrix(F(a))
        z = lambda r, c: cm.CUDAMatrix(F(np.zeros((r, c))))
        self.host = dict(x=rng.standard_normal((d, n)), w1=rng.standard_normal((d, 2 * f)) / np.sqrt(d), b1=0.1 * rng.standard_normal((2 * f, 1)),
                         w2=rng.standard_normal((f, d)) / np.sqrt(f), wv=rng.standard_normal((d, v)) / np.sqrt(d), g1=1 + 0.1 * rng.standard_normal((d, 1)),
                         c1=0.1 * rng.standard_normal((d, 1)), g2=1 + 0.1 * rng.standard_normal((d, 1)), c2=0.1 * rng.standard_normal((d, 1)),
                         labels=rng.integers(-1, v, (1, n)).astype(np.float64), lw=rng.standard_normal((1, n)), ew=0.1 * rng.standard_normal((1, n)),
                         step=np.array([[3.0]]))
        self.host = {k: F(a).astype(np.float64) for k, a in self.host.items()}
        self.m = {k: D(a) for k, a in self.host.items()}
        for name, r, c in (('h1', d, n), ('gated', f, n), ('pre', 2 * f, n), ('down', d, n), ('x2', d, n), ('h2', d, n), ('logits', v, n), ('logp', 1, n),
                           ('entropy', 1, n), ('log_z', 1, n), ('dh2', d, n), ('dx2', d, n), ('ddown', d, n), ('dgated', f, n), ('dh1', d, n),
                           ('dx', d, n), ('dw1', d, 2 * f), ('db1', 2 * f, 1), ('dw2', f, d), ('dwv', d, v), ('dg1', d, 1), ('dc1', d, 1),
                           ('dg2', d, 1), ('dc2', d, 1)):
            self.m[name] = z(r, c)

    GRADS = ('dx', 'dw1', 'db1', 'dw2', 'dwv', 'dg1', 'dc1', 'dg2', 'dc2')

    def step(self):
        cm, m = self.cm, self.m
        drop = dict(dropprob=0.25, seed=99, stream=1, step=m['step'])
        cm.layer_norm(m['x'], m['g1'], m['c1'], target=m['h1'])
        cm.dot_gated(m['w1'].T, m['h1'], m['b1'], target=m['gated'], pre=m['pre'])
        cm.dot(m['w2'].T, m['gated'], target=m['down'])
        cm.counter_dropout(m['down'], residual=m['x'], target=m['x2'], **drop)
        cm.layer_norm(m['x2'], m['g2'], m['c2'], target=m['h2'])
        cm.dot(m['wv'].T, m['h2'], target=m['logits'])
        cm.log_probs(m['logits'], m['labels'], logp=m['logp'], entropy=m['entropy'], log_z=m['log_z'])
        dlogits = cm.log_probs_grad(m['logits'], m['labels'], m['log_z'], m['lw'], m['entropy'], m['ew'])       # in place
        cm.dot(m['h2'], dlogits.T, target=m['dwv'])
        cm.dot(m['wv'], dlogits, target=m['dh2'])
        cm.layer_norm_grad(m['dh2'], m['x2'], m['g2'], target=m['dx2'], gain_grad=m['dg2'], bias_grad=m['dc2'])
        cm.counter_dropout(m['dx2'], target=m['ddown'], **drop)
        cm.dot(m['gated'], m['ddown'].T, target=m['dw2'])
        cm.dot(m['w2'], m['ddown'], target=m['dgated'])
        cm.dot_gated_grad(m['dgated'], m['w1'].T, m['h1'], m['pre'], m1_grad=m['dw1'], m2_grad=m['dh1'], bias_grad=m['db1'])
        cm.layer_norm_grad(m['dh1'], m['x'], m['g1'], target=m['dx'], gain_grad=m['dg1'], bias_grad=m['dc1'])
        m['dx'].add(m['dx2'])

    def oracle(self, h, step=3.0):
        """(objective, gradients by name) in 64 bits."""
        keep = tok.dropout_keep(h['x'].shape, 0.25, 99, 1, step) / 0.75
        h1 = tok.layer_norm(h['x'], h['g1'], h['c1'])
        gated, pre = tok.dot_gated(h['w1'].T, h1, h['b1'])
        x2 = h['x'] + keep * (h['w2'].T @ gated)
        h2 = tok.layer_norm(x2, h['g2'], h['c2'])
        logits = h['wv'].T @ h2
        o = tok.log_probs(logits, h['labels'])
        dl = tok.log_probs_grad(logits, h['labels'], o['log_z'], h['lw'], o['entropy'], h['ew'])
        g = dict(dwv=h2 @ dl.T)
        dx2, g['dg2'], g['dc2'] = tok.layer_norm_grad(h['wv'] @ dl, x2, h['g2'])
        dd = keep * dx2
        g['dw2'] = gated @ dd.T
        dp = tok.gate_grad(h['w2'] @ dd, pre)
        g['dw1'], g['db1'] = h1 @ dp.T, dp.sum(axis=1, keepdims=True)
        dx, g['dg1'], g['dc1'] = tok.layer_norm_grad(h['w1'] @ dp, h['x'], h['g1'])
        g['dx'] = dx + dx2
        return float((h['lw'] * o['logp']).sum() + (h['ew'] * o['entropy']).sum()), g, o


def test_a_block_forward_and_backward(cm, rng):
    """All of them as they are used.  Every gradient against the oracle's (rounding errors of a chain of ten operators, each about
    10 u to 100 u of the magnitudes it handles: 2e-5 of the largest entry), and along random directions against differences of
    the oracle's objective."""
    b = Block(cm, rng)
    b.step()
    value, grads, o = b.oracle(b.host)
    assert np.max(np.abs(b.m['logp'].asarray() - o['logp'])) < 1e-5 * np.max(np.abs(o['logp']))
    for name in b.GRADS:
        got, want = b.m[name].asarray(), grads[name]
        assert np.max(np.abs(got - want)) < 2e-5 * np.max(np.abs(want)), name
        where = 'x' if name == 'dx' else name[1:]
        way = rng.standard_normal(want.shape)
        ends = []
        for s in (1e-5, -1e-5):
            h = dict(b.host)
            h[where] = h[where] + s * way
            ends.append(b.oracle(h)[0])
        slope = (ends[0] - ends[1]) / 2e-5
        assert abs(np.sum(got * way) - slope) < 1e-4 * np.max(np.abs(want)) * np.sqrt(want.size) + 1e-6 * (1 + abs(value)), name


def bits(mats):
    return [m.asarray().view(np.uint32).copy() for m in mats]


def test_recorded_blocks_draw_fresh_masks(cm):
    """A recorded step, replayed with eager work and synchronisations between the replays: each replay has the bits of the step called
    with the same counter, which a call in the recording moves on."""
    a, b = Block(cm, np.random.default_rng(8)), Block(cm, np.random.default_rng(8))
    names = Block.GRADS + ('logp', 'entropy', 'x2')
    def step(o):
        o.step()
        o.m['step'].add(1.0)
    want = []
    for _ in range(5):
        step(a)
        want.append(bits(a.m[n] for n in names))
    assert any(not np.array_equal(p, q) for p, q in zip(want[0], want[1]))
    step(b)
    assert all(np.array_equal(p, q) for p, q in zip(bits(b.m[n] for n in names), want[0]))
    with cm.Graph() as g:
        step(b)
    with cm.Graph() as other:                                   # a second recording shares the library's workspaces
        step(a)
    for i in range(1, 5):
        g.launch()
        assert all(np.array_equal(p, q) for p, q in zip(bits(b.m[n] for n in names), want[i])), i
        other.launch()
        c = Block(cm, np.random.default_rng(i), d=33, f=50, v=201, n=9)
        c.step()
        c.m['dx'].asarray()


def test_a_block_on_a_stream_of_the_callers(cm):
    hip = ct.CDLL('libamdhip64.so')
    a, b = Block(cm, np.random.default_rng(9)), Block(cm, np.random.default_rng(9))
    a.step()
    want = bits(a.m[n] for n in Block.GRADS)
    stream = ct.c_void_p()
    assert hip.hipStreamCreateWithFlags(ct.byref(stream), 1) == 0
    cm.cuda_sync_threads()
    cm._cudamat.graph_set_stream(stream, 0)
    try:
        b.step()
        cm.launch_deferred()
        assert hip.hipStreamSynchronize(stream) == 0
    finally:
        cm._cudamat.graph_set_stream(None, 0)
    assert all(np.array_equal(p, q) for p, q in zip(bits(b.m[n] for n in Block.GRADS), want))
    assert hip.hipStreamDestroy(stream) == 0


def test_results_do_not_depend_on_the_run(cm, rng):
    """The same call twice: the same bits (nothing is added up in the order in which workgroups happen to come)."""
    h, w = 3000, 700
    x, dy, gain = cm.CUDAMatrix(F(rng.standard_normal((h, w)))), cm.CUDAMatrix(F(rng.standard_normal((h, w)))), cm.CUDAMatrix(F(rng.standard_normal((h, 1))))
    big, labels = cm.CUDAMatrix(F(rng.standard_normal((60000, 3)))), cm.CUDAMatrix(F([[5, 6, 7]]))
    runs = []
    for _ in range(4):
        t, gg, bg = cm.empty((h, w)), cm.empty((h, 1)), cm.empty((h, 1))
        cm.layer_norm_grad(dy, x, gain, target=t, gain_grad=gg, bias_grad=bg)
        o = [cm.empty((1, 3)) for _ in range(3)] + [cm.empty((20, 3)), cm.empty((20, 3))]
        cm.log_probs(big, labels, *o)
        runs.append(bits([t, gg, bg] + o))
    for r in runs[1:]:
        assert all(np.array_equal(p, q) for p, q in zip(r, runs[0]))


def test_more_than_two_to_the_31_entries(cm):
    """Offsets beyond 2^31 entries and 2^33 bytes: the last columns of each operator are those of the same columns by themselves."""
    h, w = 65536, 32800
    lib = cm._cudamat
    big = cm.empty((h, w))
    big.assign(0.125)
    tail = F(np.random.default_rng(4).standard_normal((h, 16)))
    small = cm.CUDAMatrix(tail)
    view = big.slice(w - 16, w)
    def reset():
        big.assign(0.125)
        view.assign(small)
    reset()
    gain, bias = cm.CUDAMatrix(F(np.full((h, 1), 1.5))), cm.CUDAMatrix(F(np.full((h, 1), -0.5)))
    want = cm.layer_norm(small, gain, bias, target=cm.empty((h, 16))).asarray().copy()
    cm.layer_norm(big, gain, bias)
    assert np.array_equal(view.asarray(), want) and (big.slice(0, 1).asarray() == -0.5).all()
    reset()
    keep = tok.dropout_keep((h, w), 0.5, 3, first=h * (w - 16), count=16 * h).reshape((h, 16), order='F')
    cm.counter_dropout(big, 0.5, 3)
    assert np.array_equal(view.asarray(), np.where(keep, 2 * tail, np.float32(0)))
    reset()
    labels = F(np.full((1, w), 7.0))
    o, s = [cm.empty((1, w)) for _ in range(3)] + [cm.empty((3, w)), cm.empty((3, w))], [cm.empty((1, 16)) for _ in range(3)] + [cm.empty((3, 16)), cm.empty((3, 16))]
    cm.log_probs(big, cm.CUDAMatrix(labels), *o)
    cm.log_probs(small, cm.CUDAMatrix(labels[:, :16]), *s)
    for a, b in zip(o, s):
        got, ref = a.asarray()[:, -16:], b.asarray()
        assert np.allclose(got, ref, rtol=1e-6)
    want = cm.log_probs_grad(small, cm.CUDAMatrix(labels[:, :16]), s[2], target=cm.empty((h, 16))).asarray().copy()
    cm.log_probs_grad(big, cm.CUDAMatrix(labels), o[2])
    assert np.max(np.abs(view.asarray() - want)) < 1e-6
    for m in [big, small, gain, bias] + o + s:
        m.free_device_memory()
