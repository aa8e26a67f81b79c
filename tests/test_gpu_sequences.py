"""Embeddings, gated recurrences along sequences and sampling of tokens through the Python entry points against their restatements in 64
bits.

Bounds, with u = 2^-24 (half a step of fp32, relative).  embed: one product, the same bits.  embed_grad: n terms in any order are off by at most
n - 1 roundings of the sum of their magnitudes; the scaling and the accumulation add 3.  gated_scan: the oracle follows how an error of one
unit of every step's magnitudes (those of the sums without cancellation) grows along the sequence; a step has the gate (2 ulp = 4 u), 1 - gate and its
product with the input (5 u), the recurrence (1 u) and, where stretches are joined, the product of gates (1 u a step) and the join (2 u): 16 in all."""
import ctypes as ct

import numpy as np
import pytest

from oracle import sequence_oracle as seq
from oracle import token_oracle as tok
from test_gpu_tokens import F, U, bits, check, device, neighbours_untouched

pytestmark = pytest.mark.gpu

STEP = 16


def frequent(rng, n, w):
    """Tokens, the first ones most frequent, and some that are none."""
    l = np.minimum((np.exp(rng.random((1, w)) * np.log(n + 1)) - 1).astype(int), n - 1).astype(np.float64)
    l[rng.random((1, w)) < 0.1] = -1
    return F(l)


# ------------------------------------------------------------------ embeddings

EMBED_SHAPES = [(1, 1, 1), (1, 7, 3), (2, 5, 9), (3, 1000, 70), (4, 17, 1), (5, 300, 2000), (63, 33, 257), (64, 1, 50000), (100, 257, 100), (255, 3, 4), (1000, 100, 40),
                (1001, 65, 33), (1024, 4, 1000), (4096, 70, 300), (4099, 31, 12), (10000, 9, 5), (70001, 3, 4), (8, 40000, 16)]


@pytest.mark.parametrize("h,w,n", EMBED_SHAPES)
@pytest.mark.parametrize("skip", [0, 1])
def test_embed(cm, rng, h, w, n, skip):
    e, labels = F(rng.standard_normal((h, n))), frequent(rng, n, w)
    for mult in (1.0, 0.37):
        y = device(cm, np.full((h, w), np.nan), skip)
        assert cm.embed(device(cm, e, skip), cm.CUDAMatrix(labels), target=y, mult=mult) is y
        want = F(seq.embed(e, labels, float(np.float32(mult))))             # (a product of two fp32 numbers is exact in fp64)
        assert np.array_equal(y.asarray(), want)
        neighbours_untouched(y, skip)
    assert np.array_equal(cm.embed(cm.CUDAMatrix(e), cm.CUDAMatrix(labels)).asarray(), F(seq.embed(e, labels)))


def test_labels_that_are_no_tokens(cm, rng):
    e = F(rng.standard_normal((6, 5)))
    labels = F([[-1, -0.5, 5, 1e30, np.nan, np.inf, -np.inf, -0.0, 4.75, 2 ** 31, -2 ** 31]])
    y = cm.embed(cm.CUDAMatrix(e), cm.CUDAMatrix(labels)).asarray()
    assert not y[:, [0, 1, 2, 3, 4, 5, 6, 9, 10]].any() and np.array_equal(y[:, [7, 8]], e[:, [0, 4]])
    g = cm.CUDAMatrix(F(np.full((6, 5), np.nan)))
    dy = F(rng.standard_normal((6, 11)))
    dy[:, [0, 1, 2, 3, 4, 5, 6, 9, 10]] = np.nan                          # what belongs to no token goes nowhere
    cm.embed_grad(cm.CUDAMatrix(dy), cm.CUDAMatrix(labels), g)
    want = np.zeros((6, 5)); want[:, 0], want[:, 4] = dy[:, 7], dy[:, 8]
    assert np.array_equal(g.asarray(), want)


def check_embed_grad(got, dy, labels, n, mult=1.0, old=None, beta=0.0):
    want, size, count = seq.embed_grad(dy, labels, n, mult)
    was = 0.0 if old is None else beta * old.astype(np.float64)
    check(got, was + want, U * ((count[None, :] + 2) * size + 3 * (np.abs(was) + np.abs(want))))


@pytest.mark.parametrize("h,w,n", EMBED_SHAPES + [(20, 5000, 1), (33, 9000, 7), (130, 3000, 300), (17, 20001, 256), (64, 3000, 40000), (1, 30000, 5), (260, 2049, 2), (1025, 40, 6), (2050, 33, 3), (306177, 3, 2), (512, 8192, 9), (512, 8193, 9), (3, 8000, 2000), (64, 600, 4096), (65, 513, 4090), (300, 512, 2048), (300, 513, 2049), (68, 4000, 1)])
@pytest.mark.parametrize("skip", [0, 1])
def test_embed_grad(cm, rng, h, w, n, skip):
    dy, labels = F(rng.standard_normal((h, w))), frequent(rng, n, w)
    d, l = device(cm, dy, skip), cm.CUDAMatrix(labels)
    g = device(cm, np.full((h, n), np.nan), skip)                          # beta = 0 reads nothing and writes everything
    assert cm.embed_grad(d, l, g) is g
    check_embed_grad(g.asarray(), dy, labels, n)
    neighbours_untouched(g, skip)
    old = F(rng.standard_normal((h, n)))
    for mult, beta in ((0.25, 1.0), (-2.0, 0.5)):
        g = device(cm, old, skip)
        cm.embed_grad(d, l, g, mult=mult, beta=beta)
        got = g.asarray()
        check_embed_grad(got, dy, labels, n, mult, old, beta)
        if beta == 1.0:                                                    # columns of other tokens are not touched
            absent = np.setdiff1d(np.arange(n), labels[labels >= 0].astype(int))
            assert np.array_equal(got[:, absent], old[:, absent])
        neighbours_untouched(g, skip)


@pytest.mark.parametrize("w", [1, 31, 32, 33, 63, 64, 65, 127, 128, 129, 200, 1000, 4097, 16385, 70000])
def test_embed_grad_of_one_frequent_token(cm, rng, w):
    """Runs of every length around the stretches that they are cut into, alone, first, last and between others."""
    h, n = 12, 1000
    dy = F(rng.standard_normal((h, w + 7)))
    for token, others in ((0, (5, 7)), (n - 1, (3, 4)), (500, (499, 501)), (77, (77, 77))):
        labels = F(np.full((1, w + 7), token))
        labels[0, rng.choice(w + 7, 3, replace=False)] = others[0]
        labels[0, rng.choice(w + 7, 3, replace=False)] = others[1]
        g = cm.embed_grad(cm.CUDAMatrix(dy), cm.CUDAMatrix(labels), cm.CUDAMatrix(F(np.full((h, n), np.nan))))
        check_embed_grad(g.asarray(), dy, labels, n)


@pytest.mark.parametrize("h,w", [(12, 2000), (12, 8192), (100, 8192), (3, 8192), (12, 8193), (12, 70000), (300, 70000), (1, 1 << 21)])
def test_embed_grad_of_a_frequent_token_adds_in_short_chains(cm, h, w):
    """2^25, where a step of fp32 is 4, and ones: added one after the other these would all be lost.  Bound: as many roundings as follow each other in the longest
    chain, and the scaling's."""
    if w <= 8192:
        teams = 16 if h > 64 else 64
        chain = -(-w // teams) + teams
    else:
        piece = 16
        while 8 * piece * piece < w:
            piece *= 2
        chain = piece + -(-w // piece)
    dy, labels = cm.empty((h, w)), cm.empty((1, w))
    dy.assign(1.0)
    labels.assign(3.0)
    for at in (0, w // 2, w - 1):
        dy.slice(at, at + 1).assign(float(1 << 25))
        g = cm.embed_grad(dy, labels, cm.CUDAMatrix(F(np.full((h, 5), np.nan)))).asarray()
        dy.slice(at, at + 1).assign(1.0)
        total = (1 << 25) + w - 1
        assert np.abs(g[:, 3] - float(total)).max() <= U * (chain + 1) * total < w / 2, (at, g[0, 3] - total)
        assert not g[:, [0, 1, 2, 4]].any()


def test_embed_of_no_vocabulary(cm):
    y = cm.CUDAMatrix(F(np.full((6, 5), np.nan)))
    cm.embed(cm.empty((6, 0)), cm.CUDAMatrix(F([[0, 1, -1, 2, 3]])), target=y)
    assert not y.asarray().any()


def test_embed_grad_of_no_columns_and_of_no_tokens(cm, rng):
    old = F(rng.standard_normal((6, 9)))
    for labels in (np.zeros((1, 0)), np.full((1, 5), -1.0)):
        dy = cm.empty((6, labels.shape[1]))
        for beta, want in ((0.0, np.zeros((6, 9))), (1.0, old), (0.5, F(0.5) * old)):
            g = cm.CUDAMatrix(old)
            cm.embed_grad(dy, cm.CUDAMatrix(F(labels)) if labels.size else cm.empty((1, 0)), g, beta=beta)
            assert np.array_equal(g.asarray(), want)


@pytest.mark.parametrize("h,n", [(6, 5000), (1030, 5000), (3, 1 << 20)])
def test_embed_grad_of_no_columns_and_many_tokens(cm, rng, h, n):
    old = F(rng.standard_normal((h, n)))
    for beta, want in ((0.0, np.zeros((h, n))), (1.0, old), (0.5, F(0.5) * old)):
        g = cm.CUDAMatrix(old)
        cm.embed_grad(cm.empty((h, 0)), cm.empty((1, 0)), g, beta=beta)
        assert np.array_equal(g.asarray(), want)


def test_embed_grad_gives_the_same_bits_every_time(cm, rng):
    h, w, n = 200, 30000, 5000
    d, l = cm.CUDAMatrix(F(rng.standard_normal((h, w)))), cm.CUDAMatrix(frequent(rng, n, w))
    runs = [bits([cm.embed_grad(d, l, cm.empty((h, n)))])[0] for _ in range(5)]
    assert all(np.array_equal(r, runs[0]) for r in runs[1:])


# ------------------------------------------------------------------ gated recurrences

def scan_inputs(rng, f, w, n):
    pre = rng.standard_normal((2 * f, w))
    pre[:f] += rng.uniform(-2, 7, (f, 1))
    return F(pre), F(rng.standard_normal((f, n))), F(rng.standard_normal((f, w))), F(rng.standard_normal((f, n)))


def check_scan(cm, rng, f, w, n, offsets=None, skip=0, states=True):
    pre, state, dy, dlast = scan_inputs(rng, f, w, n)
    at = seq.borders(w, offsets, n)
    D = lambda a: device(cm, a, skip)
    args = dict(offsets=None if offsets is None else cm.CUDAMatrix(F([offsets])), sequences=n, state=D(state) if states else None)
    y, last = D(np.full((f, w), 3.25)), D(np.full((f, n), np.nan)) if states else None
    assert cm.gated_scan(D(pre), target=y, last=last, **args) is y
    want, want_last, off, last_off = seq.gated_scan(pre, at, state if states else None)
    outside = np.isnan(want).all(axis=0)
    got = y.asarray().copy()
    assert (got[:, outside] == 3.25).all(), 'columns of no sequence'
    check(got[:, ~outside], want[:, ~outside], STEP * U * off[:, ~outside], 'y')
    if states:
        check(last.asarray(), want_last, STEP * U * last_off + U * np.abs(want_last), 'last')
        neighbours_untouched(last, skip)
    neighbours_untouched(y, skip)
    # backward, from these very columns
    dp, ds = D(np.full((2 * f, w), 3.25)), D(np.full((f, n), np.nan)) if states else None
    more = dict(args, last_deriv=D(dlast) if states else None, state_grad=ds)
    assert cm.gated_scan_grad(D(dy), D(pre), y, target=dp, **more) is dp
    want, want_state, off, state_off = seq.gated_scan_grad(dy, pre, got, at, state if states else None, dlast if states else None)
    g = dp.asarray().copy()
    assert (g[:, outside] == 3.25).all(), 'derivatives of no sequence'
    check(g[:, ~outside], want[:, ~outside], STEP * U * (off + np.abs(want))[:, ~outside], 'dpre')
    if states:
        check(ds.asarray(), want_state, STEP * U * state_off + U * np.abs(want_state), 'dstate')
        neighbours_untouched(ds, skip)
    neighbours_untouched(dp, skip)
    # in place: the derivative over pre, that of the states over last_deriv, the last columns over the states
    p = D(pre)
    if states:
        more['last_deriv'] = more['state_grad'] = D(dlast)
    cm.gated_scan_grad(D(dy), p, y, **more)
    assert np.array_equal(p.asarray()[:, ~outside], g[:, ~outside]) and np.array_equal(p.asarray()[:, outside], pre[:, outside])
    if states:
        assert np.array_equal(more['state_grad'].asarray(), ds.asarray())
        y2, s2 = D(np.full((f, w), 3.25)), args['state']
        cm.gated_scan(D(pre), target=y2, last=s2, **args)
        assert np.array_equal(s2.asarray(), last.asarray()) and np.array_equal(y2.asarray(), got)


@pytest.mark.parametrize("f,w,n", [(1, 1, 1), (1, 9, 1), (2, 3, 3), (3, 64, 2), (4, 100, 1), (5, 7, 7), (16, 500, 1), (31, 1000, 4), (64, 63, 1), (64, 64, 1), (65, 65, 1), (100, 130, 2),
                                   (128, 257, 1), (130, 4100, 1), (255, 513, 3), (256, 1024, 8), (1001, 33, 3), (2048, 4, 4), (1024, 600, 600), (7, 20000, 1), (1, 5000, 1),
                                   (12, 5000, 5000), (700, 2048, 2), (4097, 20, 1)])
@pytest.mark.parametrize("skip", [0, 1])
def test_gated_scan_and_its_gradients(cm, rng, f, w, n, skip):
    check_scan(cm, rng, f, w, n, skip=skip)
    check_scan(cm, rng, f, w, n, skip=skip, states=False)


@pytest.mark.parametrize("f,w", [(1, 300), (33, 1500), (64, 700), (130, 5000), (1026, 260)])
@pytest.mark.parametrize("skip", [0, 1])
def test_gated_scan_of_sequences_of_any_lengths(cm, rng, f, w, skip):
    for n in (1, 2, 9, 200):
        cuts = np.sort(rng.integers(0, w + 1, n + 1))
        check_scan(cm, rng, f, w, n, cuts, skip)
    lengths = np.array([0, 0, 1, 1, 63, 0, 64, 65, 1, 0, 128, 0, 0])
    check_scan(cm, rng, f, w if w > 330 else 340, len(lengths), 3 + np.concatenate([[0], np.cumsum(lengths)]), skip)
    check_scan(cm, rng, f, w, 3, [0, w, w, w], skip)
    check_scan(cm, rng, f, w, 2, [5, 5, 5], skip)
    check_scan(cm, rng, f, w, 2, [0, w // 2, w], skip, states=False)


@pytest.mark.parametrize("f,w,n", [(65606, 150, 2), (131072, 130, 1)])
def test_gated_scan_of_more_units_than_a_launch_takes(cm, rng, f, w, n):
    check_scan(cm, rng, f, w, n)


@pytest.mark.parametrize("f", [449, 512, 963, 1024, 2001])
def test_gated_scan_of_tiles_that_xcds_share(cm, rng, f):
    check_scan(cm, rng, f, 700, 3, [0, 5, 400, 699], skip=1)


@pytest.mark.parametrize("f,w,n", [(376, 814, 450), (65, 3, 1000), (20, 40, 700), (64, 700, 65), (130, 1, 64), (7, 900, 3000)])
def test_gated_scan_of_many_sequences_most_of_them_empty(cm, rng, f, w, n):
    check_scan(cm, rng, f, w, n, np.sort(rng.integers(0, w + 1, n + 1)), skip=1)
    check_scan(cm, rng, f, w, n, np.r_[[0] * (n // 2), [w] * (n + 1 - n // 2)])


def test_gated_scan_of_no_columns(cm, rng):
    state = F(rng.standard_normal((5, 3)))
    last = cm.empty((5, 3))
    cm.gated_scan(cm.empty((10, 0)), target=cm.empty((5, 0)), state=cm.CUDAMatrix(state), last=last)
    assert np.array_equal(last.asarray(), state)
    cm.gated_scan(cm.empty((10, 0)), target=cm.empty((5, 0)), last=last)
    assert not last.asarray().any()
    cm.gated_scan_grad(cm.empty((5, 0)), cm.empty((10, 0)), cm.empty((5, 0)), last_deriv=cm.CUDAMatrix(state), state_grad=last)
    assert np.array_equal(last.asarray(), state)


def test_gated_scan_step_by_step_is_the_scan(cm, rng):
    """Decoding: one column a sequence, the states in place, gives what the scan over all columns gives to rounding."""
    f, n, t = 70, 3, 40
    pre, state, _, _ = scan_inputs(rng, f, n * t, n)
    want, want_last, off, last_off = seq.gated_scan(pre, seq.borders(n * t, None, n), state)
    s = cm.CUDAMatrix(state)
    for i in range(t):
        y = cm.gated_scan(cm.CUDAMatrix(F(pre[:, i::t])), state=s, last=s)
        assert np.array_equal(y.asarray(), s.asarray())
        check(y.asarray(), want[:, i::t], STEP * U * off[:, i::t] + 1e-30, i)


@pytest.mark.parametrize("f,w", [(3, 40), (64, 3000), (130, 700)])
def test_gated_scan_keeps_infinities_and_nan_in_their_sequence(cm, rng, f, w):
    n = 4
    pre, state, dy, dlast = scan_inputs(rng, f, w, n)
    at = [0, w // 4, w // 2, 3 * w // 4, w]
    pre[f:, w // 4 + 2], pre[0, w // 2 + 1], state[:, 3] = np.nan, np.nan, np.inf
    pre[1, :w // 4] = 200.0                                             # a gate of 1: the state is kept
    pre[2, :w // 4] = -200.0                                            # of 0: it is the input
    state[:, 0] = 2.0
    y, last = cm.empty((f, w)), cm.empty((f, n))
    cm.gated_scan(cm.CUDAMatrix(pre), target=y, offsets=cm.CUDAMatrix(F([at])), state=cm.CUDAMatrix(state), last=last)
    got = y.asarray()
    finite = [c for c in range(w) if c < at[1] + 2 or at[2] <= c < at[3]]
    want, _, off, _ = seq.gated_scan(pre, at, state)
    check(got[1:, finite], want[1:, finite], (STEP * U * off)[1:, finite])
    assert (got[1, :at[1]] == 2.0).all() and np.array_equal(got[2, :at[1]], pre[f + 2, :at[1]])
    assert not np.isfinite(got[:, at[1] + 2:at[2]]).any() and not np.isfinite(got[0, at[2] + 1:at[3]]).any() and not np.isfinite(got[3:, at[3]:]).any()
    assert np.isfinite(last.asarray()[3:, [0, 2]]).all() and not np.isfinite(last.asarray()[3:, [1, 3]]).any()
    # back: what is not finite in a derivative reaches the columns before it in its sequence alone
    dy[:, at[2] - 3] = np.nan
    pre, state = scan_inputs(rng, f, w, n)[:2]
    y = cm.gated_scan(cm.CUDAMatrix(pre), offsets=cm.CUDAMatrix(F([at])), state=cm.CUDAMatrix(state))
    ds = cm.empty((f, n))
    dp = cm.gated_scan_grad(cm.CUDAMatrix(dy), cm.CUDAMatrix(pre), y, target=cm.empty((2 * f, w)), offsets=cm.CUDAMatrix(F([at])),
                            state=cm.CUDAMatrix(state), state_grad=ds).asarray()
    assert np.isnan(dp[:, at[1]:at[2] - 2]).all() and np.isfinite(dp[:, :at[1]]).all() and np.isfinite(dp[:, at[2] - 2:]).all()
    assert np.isnan(ds.asarray()[:, 1]).all() and np.isfinite(ds.asarray()[:, [0, 2, 3]]).all()


def test_offsets_out_of_place_stay_within_the_matrix(cm, rng):
    """Below 0, behind the last column, NaN: as 0 or the last column; the columns around the matrix are not touched."""
    f, w = 40, 300
    pre, state, dy, dlast = scan_inputs(rng, f, w, 3)
    y, last = device(cm, np.full((f, w), 7.25), 4), device(cm, np.zeros((f, 3)), 4)
    cm.gated_scan(cm.CUDAMatrix(pre), target=y, offsets=cm.CUDAMatrix(F([[-5, 100, 250, 1e9]])), state=cm.CUDAMatrix(state), last=last)
    want, want_last, off, last_off = seq.gated_scan(pre, [0, 100, 250, w], state)
    check(y.asarray(), want, STEP * U * off)
    check(last.asarray(), want_last, STEP * U * last_off + U * np.abs(want_last))
    for o in ([np.nan, np.inf, -np.inf, np.nan], [250, 100, 200, 50], [300, 0, 300, 0]):
        dp = device(cm, np.full((2 * f, w), 7.25), 4)
        cm.gated_scan(cm.CUDAMatrix(pre), target=y, offsets=cm.CUDAMatrix(F([o])), state=cm.CUDAMatrix(state), last=last)
        cm.gated_scan_grad(cm.CUDAMatrix(dy), cm.CUDAMatrix(pre), y, target=dp, offsets=cm.CUDAMatrix(F([o])), state=cm.CUDAMatrix(state), state_grad=last)
        for m in (y, last, dp):
            neighbours_untouched(m, 4)


@pytest.mark.parametrize("f,w,at", [(5, 40, [3, 20, 33]), (70, 900, [0, 0, 500, 899]), (64, 10, [4, 4])])
def test_a_scan_into_a_matrix_of_its_own_has_zeros_in_columns_of_no_sequence(cm, rng, f, w, at):
    """Whatever its memory held."""
    pre, state = scan_inputs(rng, f, w, len(at) - 1)[:2]
    want, _, off, _ = seq.gated_scan(pre, at, state)
    outside = np.ones(w, dtype=bool)
    outside[at[0]:at[-1]] = False
    for _ in range(3):
        was = cm.CUDAMatrix(F(np.full((f, w), np.nan)))
        was.free_device_memory()                                         # (its block is the next one of this size)
        y = cm.gated_scan(cm.CUDAMatrix(pre), offsets=cm.CUDAMatrix(F([at])), state=cm.CUDAMatrix(state))
        got = y.asarray()
        assert outside.any() and not got[:, outside].any()
        check(got[:, ~outside], want[:, ~outside], STEP * U * off[:, ~outside])
    assert cm.gated_scan(cm.empty((2 * f, 0)), offsets=cm.CUDAMatrix(F([[0, 0]]))).shape == (f, 0)


def test_gated_scan_gives_the_same_bits_every_time(cm, rng):
    f, w = 300, 9000
    pre, state, dy, _ = scan_inputs(rng, f, w, 1)
    P, S, D = cm.CUDAMatrix(pre), cm.CUDAMatrix(state), cm.CUDAMatrix(dy)
    runs = []
    for _ in range(5):
        y, ds, dp = cm.gated_scan(P, state=S), cm.empty((f, 1)), cm.empty((2 * f, w))
        cm.gated_scan_grad(D, P, y, target=dp, state=S, state_grad=ds)
        runs.append(bits([y, dp, ds]))
    for r in runs[1:]:
        assert all(np.array_equal(p, q) for p, q in zip(r, runs[0]))


def test_gated_scan_of_many_sizes_in_turn(cm):
    """What workgroups hand to each other stands where other sizes, and other launches of the same size, have left theirs: every call has the bits of
    its first one, in whatever order the sizes come, eagerly and replayed."""
    rng = np.random.default_rng(12)
    sets = []
    for f, w in ((64, 3000), (65, 2500), (300, 700), (1, 9000), (30, 40000), (200, 5000), (700, 1300), (64, 60000), (1100, 400)):
        pre, state, dy, _ = scan_inputs(rng, f, w, 1)
        s = dict(P=cm.CUDAMatrix(pre), S=cm.CUDAMatrix(state), D=cm.CUDAMatrix(dy), y=cm.empty((f, w)), dp=cm.empty((2 * f, w)), ds=cm.empty((f, 1)))
        def step(s=s):
            cm.gated_scan(s['P'], target=s['y'], state=s['S'])
            cm.gated_scan_grad(s['D'], s['P'], s['y'], target=s['dp'], state=s['S'], state_grad=s['ds'])
        step()
        s['want'] = bits([s['y'], s['dp'], s['ds']])
        want, _, off, _ = seq.gated_scan(pre[:, :300], [0, 300], state)
        check(s['y'].asarray()[:, :300], want, STEP * U * off)
        s['step'] = step
        sets.append(s)
    for s in sets:
        with cm.Graph() as g:
            s['step']()
        s['graph'] = g
    for turn in range(150):
        s = sets[int(rng.integers(len(sets)))]
        for name in ('y', 'dp', 'ds'):
            s[name].assign(7.0)
        s['graph'].launch() if turn % 3 == 0 else s['step']()
        assert all(np.array_equal(p, q) for p, q in zip(bits([s['y'], s['dp'], s['ds']]), s['want'])), turn


def rare(rng, f, w, at):
    """Inputs of a scan over very many columns in which something happens only every 400 columns or so, in one unit each: a gate of 1/2 there, of 1 elsewhere
    (sigmoid(1000), whose other side is 0), where inputs and derivatives are 0 as well.  What a stretch of columns hands on thus stays to be seen until the unit's next
    one.  Returns the inputs and the columns that the oracle has to look at: those, the ones before them and the ends of sequences."""
    n, each = len(at) - 1, 400
    pre, dy = np.zeros((2 * f, w), dtype=np.float32), np.zeros((f, w), dtype=np.float32)
    pre[:f] = 1000.0
    events = np.minimum(np.arange(0, w, each) + rng.integers(0, each, -(-w // each)), w - 1)
    units = rng.integers(0, f, events.size)
    pre[units, events], pre[f + units, events] = 0.0, rng.standard_normal(events.size)
    dy[units, events] = rng.standard_normal(events.size)
    at = np.asarray(at)
    cols = np.unique(np.concatenate([events, events - 1, at[:-1], at[1:] - 1]))
    return F(pre), F(rng.standard_normal((f, n))), F(dy), F(rng.standard_normal((f, n))), cols[(cols >= at[0]) & (cols < at[-1])]


@pytest.mark.parametrize("f,w,at", [(64, 20011, None), (130, 40000, None), (30, 40000, None), (1, 80000, None), (64, 530000, None), (20, 530000, None), (64, 20011, [5, 700, 700, 9000, 19711]),
                                    (130, 40000, [0, 3, 12345, 39990, 40000]), (30, 40000, [0, 17000, 40000]), (1, 80000, [100, 101, 9000, 79990]), (64, 530000, [9, 300000, 529000]),
                                    (7, 1060000, [0, 12345, 1060000])])
def test_gated_scan_hands_on_through_many_chunks(cm, rng, f, w, at):
    """More than 256 chunks, and more than 4096, so that links of 16 chunks, of 256 and of 4096 are joined: every column, the states and all derivatives.  Of gates of 1 and
    inputs of 0 the links are joined exactly; other joins round what `off` counts for the columns that the links are of, damped by the gates behind them, but for those
    that come last: at most three of each of four levels and two of the workgroup's own, less than 16 of the magnitudes at the last column where anything happened."""
    at = at or [0, w]
    pre, state, dy, dlast, cols = rare(rng, f, w, at)
    few = np.searchsorted(cols, at)
    o, S = cm.CUDAMatrix(F([at])), cm.CUDAMatrix(state)
    P, y, last = cm.CUDAMatrix(pre), cm.CUDAMatrix(F(np.zeros((f, w)))), cm.CUDAMatrix(F(np.zeros(state.shape)))
    cm.gated_scan(P, target=y, offsets=o, state=S, last=last)
    got = y.asarray().copy()
    want, want_last, off, last_off = seq.gated_scan(pre[:, cols], few, state)
    inside = np.arange(at[0], at[-1])
    seen = np.searchsorted(cols, inside, side='right') - 1                # (the first column of a sequence is one of them)
    check(got[:, inside], want[:, seen], (STEP + 16) * U * off[:, seen], 'y')
    assert not got[:, :at[0]].any() and not got[:, at[-1]:].any()
    check(last.asarray(), want_last, (STEP + 16) * U * last_off + U * np.abs(want_last), 'last')
    D, ds = cm.CUDAMatrix(dy), cm.CUDAMatrix(F(np.zeros(state.shape)))
    dp = cm.CUDAMatrix(F(np.zeros((2 * f, w))))
    cm.gated_scan_grad(D, P, y, target=dp, offsets=o, state=S, last_deriv=cm.CUDAMatrix(dlast), state_grad=ds)
    want, want_state, off, state_off = seq.gated_scan_grad(dy[:, cols], pre[:, cols], got[:, cols], few, state, dlast)
    g = dp.asarray()
    check(g[:, cols], want, (STEP + 16) * U * (off + np.abs(want)), 'dpre')
    rest = np.ones(w, dtype=bool)
    rest[cols] = False
    assert not g[:, rest].any()                                            # (1 - gate is 0)
    check(ds.asarray(), want_state, (STEP + 16) * U * state_off + U * np.abs(want_state), 'dstate')
    assert np.abs(want_state).max() > 0.1 and np.abs(want_last).max() > 0.1
    release(P, y, D, dp)


def test_gated_scan_gradients_against_differences(cm):
    """The device's gradients along random directions against differences of the oracle's recurrence."""
    rng = np.random.default_rng(6)
    f, w, n = 5, 60, 4
    at = [0, 20, 21, 40, 60]
    pre, state, dy, dlast = scan_inputs(rng, f, w, n)
    o = cm.CUDAMatrix(F([at]))
    y = cm.gated_scan(cm.CUDAMatrix(pre), offsets=o, state=cm.CUDAMatrix(state))
    dp, ds = cm.empty((2 * f, w)), cm.empty((f, n))
    cm.gated_scan_grad(cm.CUDAMatrix(dy), cm.CUDAMatrix(pre), y, target=dp, offsets=o, state=cm.CUDAMatrix(state), last_deriv=cm.CUDAMatrix(dlast), state_grad=ds)
    def value(p, s):
        out, last = seq.gated_scan(p, at, s)[:2]
        return np.sum(dy.astype(np.float64) * out) + np.sum(dlast.astype(np.float64) * last)
    for got, which in ((dp.asarray(), 0), (ds.asarray(), 1)):
        way = rng.standard_normal(got.shape)
        ends = [value(pre + s * way, state) if which == 0 else value(pre.astype(np.float64), state + s * way) for s in (1e-5, -1e-5)]
        assert abs(np.sum(got * way) - (ends[0] - ends[1]) / 2e-5) < 1e-5 * np.abs(got).max() * np.sqrt(got.size)


# ------------------------------------------------------------------ sampling

def check_sample(cm, x, u, skip=0, **rule):
    """Tokens have to be equal; log probabilities are rounded once from sums of weights that are whole multiples of 2^-45 (2^-38 at the tallest)
    of the greatest one."""
    h, w = x.shape
    tokens, logp = cm.CUDAMatrix(F(np.full((1, w), np.nan))), cm.CUDAMatrix(F(np.full((1, w), np.nan)))
    given = {k: cm.CUDAMatrix(F(np.reshape(v, (1, w)))) if np.ndim(v) else v for k, v in rule.items()}
    mat = device(cm, x, skip)
    cm.sample_tokens(mat, cm.CUDAMatrix(F(np.reshape(u, (1, w)))), target=tokens, logp=logp, **given)
    cm.sample_tokens(mat, cm.CUDAMatrix(F(np.reshape(u, (1, w)))), target=(again := cm.empty((1, w))), **given)
    got, got_logp = tokens.asarray()[0], logp.asarray()[0]
    assert np.array_equal(again.asarray()[0], got), 'without logp'
    for c in range(w):
        own = {k: v[c] if np.ndim(v) else v for k, v in rule.items()}
        token, lp, kept = seq.sample_token(x[:, c], u[c], **own)
        if got[c] != token and own.get('top_p', 1.0) < 1:
            # Every weight is rounded by at most half of 2^-45 (h of up to 2^17), so their sum, which is 1 or more, by at most h 2^-46 of itself, and so is a
            # border in it: where top_p of the sum is the weight of some first entries to within that (75 of 100 equal ones and 600 of
            # 4e-15 each, which are 0 as multiples, with top_p = 0.75), one entry more or less is kept.
            assert h <= 1 << 17
            for p in (1 - h * 2.0 ** -46, 1 + h * 2.0 ** -46):
                near = seq.sample_token(x[:, c], u[c], part=p, **own)
                if near[0] == got[c]:
                    token, lp, kept = near
        assert got[c] == token, (c, got[c], token, lp, len(kept), u[c], {k: v[c] if np.ndim(v) else v for k, v in rule.items()})
        assert got_logp[c] == lp or (np.isnan(lp) and np.isnan(got_logp[c])) or abs(got_logp[c] - lp) <= 2 * U * abs(lp) + 1e-10, (c, got_logp[c], lp)


SAMPLE_SHAPES = [(1, 3), (2, 9), (3, 5), (4, 8), (10, 20), (63, 4), (64, 4), (65, 5), (255, 4), (257, 9), (1000, 16), (1023, 3), (1024, 8), (1025, 5), (2047, 2), (4096, 4), (4099, 5),
                 (16384, 3), (16387, 2), (32768, 2), (32771, 3), (50000, 2), (65536, 2), (65541, 2), (131072, 2), (200003, 2)]
RULES = [dict(), dict(temperature=0.6), dict(temperature=3.0), dict(temperature=0.0), dict(top_k=1), dict(top_k=7), dict(top_k=50, top_p=0.9), dict(top_k=400), dict(top_p=0.3),
         dict(top_p=0.95), dict(top_p=0.999), dict(min_p=0.05), dict(min_p=0.2, top_p=0.8), dict(temperature=0.7, top_k=40, top_p=0.95, min_p=0.02),
         dict(temperature=1.3, top_k=1000, top_p=0.7, min_p=0.001)]


@pytest.mark.parametrize("h,w", SAMPLE_SHAPES)
@pytest.mark.parametrize("skip", [0, 1])
def test_sample_tokens(cm, rng, h, w, skip):
    x = F(rng.standard_normal((h, w)) * rng.uniform(0.3, 4.0, (1, w)))
    for rule in RULES if h < 40000 else RULES[::2]:
        check_sample(cm, x, F(rng.random(w)), skip, **rule)


@pytest.mark.parametrize("h,w", [(50, 200), (1000, 100), (5000, 40), (40000, 12), (140000, 6)])
def test_every_column_has_its_own_rule(cm, rng, h, w):
    x = F(rng.standard_normal((h, w)) * rng.uniform(0.2, 4.0, (1, w)))
    rule = dict(temperature=F(rng.choice([0.0, 0.3, 1.0, 1.7, -1.0], w)), top_k=F(rng.choice([0, 1, 2, 5, 50, h - 1, h, h + 5, 0.5, 3.9], w)),
                top_p=F(rng.choice([0.0, 0.1, 0.5, 0.9, 1.0, 2.0, -1.0], w)), min_p=F(rng.choice([0.0, 0.01, 0.3, 1.0, 5.0, -1.0], w)))
    check_sample(cm, x, F(rng.random(w)), **rule)
    check_sample(cm, x, F(rng.random(w)), temperature=rule['temperature'], top_p=0.9)
    nan = F(np.full(w, np.nan))                                          # no limits; a temperature that is none takes the greatest
    check_sample(cm, x, F(rng.random(w)), top_k=nan, top_p=nan, min_p=nan)
    tokens = cm.sample_tokens(cm.CUDAMatrix(x), cm.CUDAMatrix(F(rng.random((1, w)))), temperature=cm.CUDAMatrix(F(nan.reshape(1, w))))
    assert np.array_equal(tokens.asarray()[0], x.argmax(axis=0))


@pytest.mark.parametrize("h", [1, 2, 3, 5, 64, 100, 1000, 5000, 40000, 140000])
def test_sample_tokens_of_ties_masks_and_special_columns(cm, rng, h):
    lowest = float(np.finfo(np.float32).min)
    cols = []
    add = lambda c: cols.append(F(c).reshape(h))
    add(np.zeros(h)); add(np.full(h, -1e30)); add(np.full(h, lowest)); add(np.full(h, -np.inf)); add(np.full(h, np.inf))
    a = rng.standard_normal(h); a[h // 2] = np.nan; add(a)
    a = rng.standard_normal(h); a[h - 1] = np.inf; add(a)
    a = np.full(h, -np.inf); a[h - 1] = -3.0; add(a)
    a = np.full(h, lowest); a[h // 3] = 1.0; add(a)
    a = np.where(rng.random(h) < 0.3, -np.inf, rng.standard_normal(h)); a[0] = 0.5; add(a)
    add(rng.integers(0, 3, h)); add(np.where(np.arange(h) % 2, 0.0, -0.0)); add(np.where(np.arange(h) % 5, -1e9, 2.0))
    add(1e-30 * rng.standard_normal(h)); add(1e30 * rng.standard_normal(h)); add(-np.arange(h) / 16.0)
    x = np.stack(cols, axis=1)
    w = x.shape[1]
    few = range(w) if h <= 5000 else range(0, w, 1)
    for rule in (dict(), dict(top_k=2), dict(top_k=max(1, h // 2)), dict(top_p=0.5), dict(top_p=0.75, top_k=4), dict(min_p=1.0), dict(top_p=0.0), dict(temperature=0.0),
                 dict(temperature=1e-30), dict(temperature=float('inf')), dict(temperature=1e30, top_k=3), dict(top_p=0.4, min_p=0.5)):
        for u in (np.zeros(w), F(rng.random(w)), np.full(w, 1.0 - 2.0 ** -24)):
            check_sample(cm, x[:, few], u[few], **rule)
    u = F(np.array([np.nan, -1.0, 1.0, 7.0] * 4))
    check_sample(cm, F(np.tile(np.log([[3.0], [1.0], [2.0]]), (1, 16))), u)


@pytest.mark.parametrize("h,w", [(4097, 300), (9001, 257), (16384, 260)])
def test_limits_in_more_columns_than_compute_units(cm, rng, h, w):
    x = F(rng.standard_normal((h, w)) * rng.uniform(0.3, 4.0, (1, w)))
    x[:, 5], x[: h // 2, 7] = F(np.arange(h) % 3), -np.inf
    few = np.r_[0:9, w - 1]
    for rule in (dict(top_k=40), dict(top_k=300, top_p=0.9), dict(top_k=h // 2), dict(top_p=0.9), dict(min_p=0.05)):
        u = F(rng.random(w))
        tokens, logp = cm.empty((1, w)), cm.empty((1, w))
        cm.sample_tokens(cm.CUDAMatrix(x), cm.CUDAMatrix(F(u.reshape(1, w))), target=tokens, logp=logp, **rule)
        for c in few:
            token, lp, _ = seq.sample_token(x[:, c], u[c], **rule)
            assert tokens.asarray()[0, c] == token and abs(logp.asarray()[0, c] - lp) <= 2 * U * abs(lp) + 1e-10, (c, rule)


@pytest.mark.parametrize("h", [700, 3000, 20000])
def test_sample_tokens_of_distances_that_overflow(cm, rng, h):
    far, rows = 3e38, np.arange(h)
    x = np.stack([np.where(rows % 2, -far, far), np.where(rows % 5, far, -far + rows / h * 1e38), np.where(rows % 7, -far * (0.1 + 0.8 * rows / h), far), np.where(rows == 3, far, -far),
                  rng.uniform(-far, far, h)], axis=1)
    w = x.shape[1]
    for temperature in (float('inf'), 3e38, 1e38, 1e37):
        for rule in (dict(top_p=0.45), dict(top_p=0.75), dict(top_p=0.98), dict(top_k=h - 5), dict(top_k=100, top_p=0.9), dict(min_p=0.3), dict()):
            check_sample(cm, F(x), F(rng.random(w)), temperature=temperature, **rule)


def test_sample_tokens_of_no_rows(cm):
    logp = cm.CUDAMatrix(F([[5.0, 5.0]]))
    t = cm.sample_tokens(cm.empty((0, 2)), cm.CUDAMatrix(F([[0.5, 0.5]])), logp=logp)
    assert (t.asarray() == -1).all() and not logp.asarray().any()


def test_sample_tokens_draws_by_the_shares(cm):
    """Whatever the number: the shares of 40000 draws."""
    rng = np.random.default_rng(10)
    n, p = 40000, np.array([0.5, 0.25, 0.125, 0.0625, 0.0625])
    x = cm.CUDAMatrix(F(np.tile(np.log(p)[:, None], (1, n))))
    t = cm.sample_tokens(x, cm.CUDAMatrix(F(rng.random((1, n))))).asarray()[0].astype(int)
    assert np.max(np.abs(np.bincount(t, minlength=5) / n - p)) < 5 * np.sqrt(0.25 / n)
    t = cm.sample_tokens(x, cm.CUDAMatrix(F(rng.random((1, n)))), top_k=2).asarray()[0].astype(int)
    assert t.max() == 1 and abs(np.mean(t == 0) - 2 / 3) < 5 * np.sqrt(0.25 / n)


def test_sample_tokens_from_logits_in_a_narrow_band(cm, rng):
    """Many entries close together, equal ones among them, and borders in the middle of them."""
    for h, step in ((3000, 1e-3), (40000, 1e-4), (40000, 2.0 ** -24), (140000, 1e-5)):
        x = F(1.0 + step * rng.integers(0, 7, (h, 8)))
        for rule in (dict(top_k=h // 3), dict(top_p=0.45), dict(top_k=h // 2, top_p=0.45, min_p=0.5), dict(top_k=5)):
            check_sample(cm, x, F(rng.random(8)), **rule)


@pytest.mark.parametrize("h,w", [(36865, 1), (45057, 3), (65537, 128), (163841, 5), (266240, 2), (262145, 1), (1050000, 1), (33000, 129), (200000, 65)])
def test_sample_tokens_of_divided_columns(cm, rng, h, w):
    """Few tall columns are divided among workgroups: parts of one row, parts that end with the column, rules of every kind in one call."""
    x = F(rng.standard_normal((h, w)) * rng.uniform(0.5, 4.0, (1, w)))
    x[:, 0] = F(np.where(rng.random(h) < 0.4, -np.inf, x[:, 0]))
    x[h - 1, w - 1] = 40.0                                               # (nearly all of it, in the last row)
    few = np.unique(np.concatenate([np.arange(min(w, 3)), [w - 1]]))
    u = F(rng.random(w))
    def call(cols=None, **rule):
        given = {k: cm.CUDAMatrix(F(np.reshape(v, (1, w)))) if np.ndim(v) else v for k, v in rule.items()}
        tokens, logp = cm.empty((1, w)), cm.empty((1, w))
        cm.sample_tokens(cm.CUDAMatrix(x), cm.CUDAMatrix(F(u.reshape(1, w))), target=tokens, logp=logp, **given)
        for c in few:
            token, lp, _ = seq.sample_token(x[:, c], u[c], **{k: v[c] if np.ndim(v) else v for k, v in rule.items()})
            assert tokens.asarray()[0, c] == token and abs(logp.asarray()[0, c] - lp) <= 2 * U * abs(lp) + 1e-9, (c, rule)
    call()
    call(temperature=0.0)
    call(top_k=30)
    call(top_k=900, top_p=0.9)
    call(top_k=3000)
    call(top_p=0.8, min_p=1e-4)
    kinds = rng.permutation(np.resize(np.arange(6), w))
    call(temperature=F(np.where(kinds == 0, 0.0, 0.9)), top_k=F(np.where(kinds == 1, 20, np.where(kinds == 2, 2000, 0))), top_p=F(np.where(kinds == 3, 0.7, 1.0)),
         min_p=F(np.where(kinds == 4, 0.01, 0.0)))


def test_sample_tokens_divided_and_special_columns(cm, rng):
    h = 140000
    x = F(rng.standard_normal((h, 6)))
    x[h // 2, 0], x[h - 1, 1], x[:, 2] = np.nan, np.inf, -np.inf
    x[:, 3] = -np.inf
    x[70000, 3] = -5.0
    for rule in (dict(), dict(temperature=0.0), dict(top_p=0.5), dict(top_k=3), dict(top_k=5000)):
        check_sample(cm, x, F(rng.random(6)), **rule)


def test_recorded_sampling_of_divided_columns(cm, rng):
    """Two recordings and eager calls share the workspace, which grows in between."""
    sizes = [(140000, 3, dict(top_p=0.9)), (60000, 20, dict(top_k=2000, temperature=0.8))]
    mats, nums, outs, want, graphs = [], [], [], [], []
    for h, w, rule in sizes:
        mats.append(cm.CUDAMatrix(F(rng.standard_normal((h, w)))))
        nums.append(cm.CUDAMatrix(F(rng.random((1, w)))))
        outs.append((cm.empty((1, w)), cm.empty((1, w))))
    def call(i):
        cm.sample_tokens(mats[i], nums[i], target=outs[i][0], logp=outs[i][1], **sizes[i][2])
    for i in (0, 1):
        call(i)
        want.append(bits(outs[i]))
        with cm.Graph() as g:
            call(i)
        graphs.append(g)
    big = cm.CUDAMatrix(F(rng.standard_normal((40000, 120))))
    for turn in range(4):
        for i in (0, 1, 0):
            for o in outs[i]:
                o.assign(-7)
            graphs[i].launch()
            assert all(np.array_equal(p, q) for p, q in zip(bits(outs[i]), want[i]))
        cm.sample_tokens(big, cm.CUDAMatrix(F(rng.random((1, 120)))), target=cm.empty((1, 120)), top_p=0.5)
        call(turn % 2)
        assert all(np.array_equal(p, q) for p, q in zip(bits(outs[turn % 2]), want[turn % 2]))


# ------------------------------------------------------------------ large

def test_columns_beyond_two_to_the_31_entries(cm, rng):
    """Offsets beyond 2^31 entries and 2^33 bytes."""
    h, w = 65536, 32800
    big = cm.empty((h, w))
    big.assign(0.125)
    tail = F(rng.standard_normal((h, 4)))
    big.slice(w - 4, w).assign(cm.CUDAMatrix(tail))
    y = cm.embed(big, cm.CUDAMatrix(F([[w - 1, 0, w - 4, w]])), mult=2.0).asarray()
    assert np.array_equal(y[:, [0, 2]], 2 * tail[:, [3, 0]]) and (y[:, 1] == 0.25).all() and not y[:, 3].any()
    cm.embed_grad(cm.CUDAMatrix(tail), cm.CUDAMatrix(F([[w - 1, 3, w - 1, w - 2]])), big, beta=1.0)
    got = big.slice(w - 4, w).asarray()
    assert np.array_equal(got[:, 2], tail[:, 2] + tail[:, 3]) and np.max(np.abs(got[:, 3] - (tail[:, 3] + (tail[:, 0] + tail[:, 2])))) < 1e-5
    assert np.array_equal(big.slice(3, 4).asarray()[:, 0], F(0.125) + tail[:, 1]) and (big.slice(4, 6).asarray() == 0.125).all()
    n = 3
    u = F(rng.random((1, w)))
    top = big.slice(w - n, w).asarray().copy()
    t = cm.sample_tokens(big, cm.CUDAMatrix(u), top_k=20).asarray()[0, w - n:]
    assert [int(v) for v in t] == [seq.sample_token(top[:, i], u[0, w - n + i], top_k=20)[0] for i in range(n)]


def test_more_columns_than_a_launch_takes(cm, rng):
    """Calls of several launches: the columns around their borders."""
    w = (1 << 24) + 1000
    x, u = cm.empty((2, w)), cm.empty((1, w))
    x.assign(0.0)
    u.assign(0.25)
    u.slice(w - 1001, w - 999).assign(0.75)
    u.slice(w - 3, w).assign(0.75)
    t = cm.sample_tokens(x, u).asarray()[0]
    assert t.sum() == 5 and (t[-3:] == 1).all() and (t[w - 1001:w - 999] == 1).all()
    w = (1 << 30) + 5                                                       # three rows: columns beyond 2^31 rows go into another launch
    e, labels, y = cm.CUDAMatrix(F(rng.standard_normal((3, 4)))), cm.empty((1, w)), cm.empty((3, w))
    labels.assign(2.0)
    tail = F([[0, 1, -1, 3] * 5])
    at = (1 << 31) // 3 - 10
    labels.slice(at, at + 20).assign(cm.CUDAMatrix(tail))
    labels.slice(w - 20, w).assign(cm.CUDAMatrix(tail))
    cm.embed(e, labels, target=y)
    for a in (at, w - 20):
        assert np.array_equal(y.slice(a, a + 20).asarray(), F(seq.embed(e.asarray(), tail)))
    for a in (0, at - 20, at + 20, w - 40):
        assert np.array_equal(y.slice(a, a + 20).asarray(), np.tile(e.asarray()[:, 2:3], (1, 20)))


MANY_ROWS = (1 << 31) - 2                                                   # (a multiple of 6; no multiple of 4)


def tall(cm, rng, w):
    """MANY_ROWS x w, column c holding (c + 1) / 8 and random numbers at its first, some middle and its last six rows: the matrix, and those (18 x w)."""
    big, part = cm.empty((MANY_ROWS, w)), F(rng.standard_normal((18, w)))
    for c in range(w):
        big.slice(c, c + 1).assign((c + 1) / 8)
        for at, rows in zip(tall_places(), np.split(part[:, c:c + 1], 3)):
            src = cm.CUDAMatrix(F(rows.T))
            tall_rows(big, c, at).assign(src)
            src.free_device_memory()
    return big, part


def tall_places():
    return 0, 1 << 30, MANY_ROWS - 6


def tall_rows(big, c, at, n=6):
    """Rows [at, at + n) of a column of a tall matrix, on the device."""
    rows = big.slice(c, c + 1)
    rows.reshape((1, MANY_ROWS))
    return rows.slice(at, at + n)


def tall_read(big, c):
    """What `tall` returns of a column, and whether those between are all alike (their value)."""
    part = np.concatenate([tall_rows(big, c, at).asarray().ravel() for at in tall_places()])
    rest = [tall_rows(big, c, at, 1000).asarray() for at in (6, (1 << 30) - 1000, (1 << 30) + 6, MANY_ROWS - 1006)]
    assert all((r == rest[0][0, 0]).all() for r in rest)
    return part, rest[0][0, 0]


def release(*mats):
    for m in mats:
        m.free_device_memory()


def test_embed_of_nearly_two_to_the_31_rows(cm, rng):
    e, part = tall(cm, rng, 2)
    y = cm.empty((MANY_ROWS, 5))
    y.assign(-7.0)
    cm.embed(e, cm.CUDAMatrix(F([[1, -1, 0, 1, 1]])), target=y, mult=2.0)
    for c, t in enumerate((1, -1, 0, 1, 1)):
        got, rest = tall_read(y, c)
        assert np.array_equal(got, 2 * part[:, t] if t >= 0 else np.zeros(18)) and rest == (t + 1) / 4, c
    release(e, y)


def test_embed_grad_of_nearly_two_to_the_31_rows(cm, rng):
    """Bound: three roundings of sums below 20."""
    dy, part = tall(cm, rng, 3)
    for labels, beta in (([1, 1, 0], 0.0), ([1, -1, 1], 1.0)):
        g, old = tall(cm, rng, 2)
        cm.embed_grad(dy, cm.CUDAMatrix(F([labels])), g, mult=2.0, beta=beta)
        for t in (0, 1):
            of = [c for c in range(3) if labels[c] == t]
            got, rest = tall_read(g, t)
            assert np.max(np.abs(got - (beta * old[:, t] + 2 * part[:, of].sum(axis=1)))) < 3 * U * 20 and rest == beta * (t + 1) / 8 + sum((c + 1) / 4 for c in of), (labels, t)
        release(g)
    release(dy)


def test_embed_grad_of_nearly_two_to_the_31_columns(cm, rng):
    """Whole numbers: exact.  Nearly all columns have one token, or none."""
    w = (1 << 31) - 1
    dy, labels = cm.empty((1, w)), cm.empty((1, w))
    dy.assign(0.0)
    tail = F([np.arange(1, 9)])
    for at in (0, 1 << 30, w - 8):
        dy.slice(at, at + 8).assign(cm.CUDAMatrix(tail))
    for rest in (1.0, -1.0):
        labels.assign(rest)
        for at in (0, 1 << 30, w - 8):
            labels.slice(at, at + 8).assign(cm.CUDAMatrix(F([[0, 1, 1, 0, rest, 0, 0, rest]])))
        g = cm.CUDAMatrix(F([[-1, -1, -1]]))
        cm.embed_grad(dy, labels, g, beta=1.0)
        want = np.zeros(3)
        for at in (0, 1, 2):
            for c, t in enumerate([0, 1, 1, 0, rest, 0, 0, rest]):
                if t >= 0:
                    want[int(t)] += c + 1
        assert np.array_equal(g.asarray()[0], want - 1), rest
    release(dy, labels)


def test_scans_beyond_two_to_the_31_entries(cm, rng):
    f, w = 4096, (1 << 18) + 300                                           # pre has 2^31 entries and more
    pre, y, o = cm.empty((2 * f, w)), cm.empty((f, w)), [0, 100, w - 200, w]
    pre.assign(0.5)
    p, _, d, _ = scan_inputs(rng, f, 200, 1)
    pre.slice(w - 200, w).assign(cm.CUDAMatrix(p))
    last = cm.empty((f, 3))
    cm.gated_scan(pre, target=y, offsets=cm.CUDAMatrix(F([o])), last=last)
    got = y.slice(w - 200, w).asarray().copy()
    want, _, off, _ = seq.gated_scan(p, [0, 200])
    check(got, want, STEP * U * off)
    assert np.array_equal(last.asarray()[:, 2], got[:, -1]) and np.max(np.abs(last.asarray()[:, 1] - 0.5)) < 1e-6
    dy = cm.empty((f, w))
    dy.assign(0.0)
    dy.slice(w - 200, w).assign(cm.CUDAMatrix(d))
    cm.gated_scan_grad(dy, pre, y, offsets=cm.CUDAMatrix(F([o])))
    want, _, off, _ = seq.gated_scan_grad(d, p, got, [0, 200])
    check(pre.slice(w - 200, w).asarray(), want, STEP * U * (off + np.abs(want)))
    assert not pre.slice(w - 300, w - 200).asarray().any()


def test_scans_of_more_columns_than_a_launch_takes(cm, rng):
    """Four lanes a column: 2^32 of them go into two launches, the second one from column 2^30 - 256 on.  Gates of 1 hand on what comes, and inputs and derivatives
    of 0 add nothing, so the oracle sees the other columns alone."""
    w, n = (1 << 30) + 1000, 40
    places = (0, (1 << 30) - 256 - n // 2, w - n)
    pre, y, dy = cm.empty((2, w)), cm.empty((1, w)), cm.empty((1, w))
    pre.assign(1000.0)
    dy.assign(0.0)
    p, state, d, dlast = scan_inputs(rng, 1, 3 * n, 1)
    for i, at in enumerate(places):
        pre.slice(at, at + n).assign(cm.CUDAMatrix(F(p[:, n * i:n * i + n])))
        dy.slice(at, at + n).assign(cm.CUDAMatrix(F(d[:, n * i:n * i + n])))
    last = cm.empty((1, 1))
    cm.gated_scan(pre, target=y, state=cm.CUDAMatrix(state), last=last)
    got = np.concatenate([y.slice(at, at + n).asarray() for at in places], axis=1)
    want, want_last, off, last_off = seq.gated_scan(p, [0, 3 * n], state)
    check(got, want, STEP * U * off)
    assert last.asarray()[0, 0] == got[0, -1]
    # What is handed on was joined from the links of one or two chunks and of what came before them, not added up column by column: at most 4 joins, each a
    # rounding of what `off` has counted once at that column.  Links of gates of 1 and sums of 0 are joined exactly.
    for i, (a, b) in enumerate(zip(places, places[1:])):
        at = n * i + n - 1
        for c in [c for c in (a + n, (a + b) // 2, b - 1000) if c + 1000 <= b]:
            assert (np.abs(y.slice(c, c + 1000).asarray() - want[0, at]) <= (STEP + 4) * U * off[0, at]).all(), (i, c)
    ds = cm.empty((1, 1))
    cm.gated_scan_grad(dy, pre, y, state=cm.CUDAMatrix(state), last_deriv=cm.CUDAMatrix(dlast), state_grad=ds)
    want, want_state, off, state_off = seq.gated_scan_grad(d, p, got, [0, 3 * n], state, dlast)
    check(np.concatenate([pre.slice(at, at + n).asarray() for at in places], axis=1), want, STEP * U * (off + np.abs(want)))
    check(ds.asarray(), want_state, STEP * U * state_off + U * np.abs(want_state))
    assert not pre.slice(n, n + 1000).asarray().any() and not pre.slice(places[1] - 1000, places[1]).asarray().any()
    release(pre, y, dy)


def test_scans_without_columns_and_states_of_more_entries_than_a_launch_takes(cm, rng):
    f, n = 1 << 21, (1 << 11) + 1
    state, last, tail = cm.empty((f, n)), cm.empty((f, n)), F(rng.standard_normal((f, 2)))
    state.assign(0.5)
    last.assign(-1.0)
    state.slice(n - 2, n).assign(cm.CUDAMatrix(tail))
    cm.gated_scan(cm.empty((2 * f, 0)), target=cm.empty((f, 0)), state=state, last=last)
    assert np.array_equal(last.slice(n - 2, n).asarray(), tail)
    assert all((last.slice(c, c + 1).asarray() == 0.5).all() for c in (0, n // 2, n - 3))
    cm.gated_scan_grad(cm.empty((f, 0)), cm.empty((2 * f, 0)), cm.empty((f, 0)), state_grad=last, sequences=n)
    assert not any(last.slice(c, c + 1).asarray().any() for c in (0, n // 2, n - 3, n - 2, n - 1))
    release(state, last)


# ------------------------------------------------------------------ together

class Net(object):
    """A net over tokens of packed texts: embedding, norm, gated recurrence, gated product onto the residual, logits by the table itself, log
    probabilities; and back to every weight and to the states that the texts begin with."""

    def __init__(self, cm, rng, d=60, f=48, v=500, at=(0, 40, 41, 41, 100), pad=7):
        self.cm, self.at, self.w = cm, list(at), at[-1] + pad
        n = len(at) - 1
        labels = rng.integers(0, v, (1, self.w)).astype(np.float64)
        labels[0, at[-1]:] = -1
        aims = np.where(labels >= 0, rng.integers(0, v, (1, self.w)), -1)
        self.host = dict(e=0.3 * rng.standard_normal((d, v)), labels=labels, aims=aims, g=1 + 0.1 * rng.standard_normal((d, 1)), c=0.1 * rng.standard_normal((d, 1)),
                         w1=rng.standard_normal((d, 2 * f)) / np.sqrt(d), w2=rng.standard_normal((f, 2 * d)) / np.sqrt(f), b2=0.1 * rng.standard_normal((2 * d, 1)),
                         state=rng.standard_normal((f, n)), lw=rng.standard_normal((1, self.w)))
        self.host = {k: F(a).astype(np.float64) for k, a in self.host.items()}
        self.m = {k: cm.CUDAMatrix(F(a)) for k, a in self.host.items()}
        self.m['offsets'] = cm.CUDAMatrix(F([self.at]))
        w = self.w
        for name, r, c in (('x', d, w), ('h', d, w), ('pre', 2 * f, w), ('s', f, w), ('last', f, n), ('halves', 2 * d, w), ('y', d, w), ('logits', v, w), ('logp', 1, w), ('log_z', 1, w),
                           ('dy', d, w), ('ds', f, w), ('dh', d, w), ('dx', d, w), ('de', d, v), ('dg', d, 1), ('dc', d, 1), ('dw1', d, 2 * f), ('dw2', f, 2 * d), ('db2', 2 * d, 1),
                           ('dstate', f, n)):
            self.m[name] = cm.CUDAMatrix(F(np.zeros((r, c))))

    GRADS = ('de', 'dg', 'dc', 'dw1', 'dw2', 'db2', 'dstate')

    def step(self):
        cm, m = self.cm, self.m
        packed = dict(offsets=m['offsets'], state=m['state'])
        cm.embed(m['e'], m['labels'], target=m['x'], mult=2.0)
        cm.layer_norm(m['x'], m['g'], m['c'], target=m['h'])
        cm.dot(m['w1'].T, m['h'], target=m['pre'])
        cm.gated_scan(m['pre'], target=m['s'], last=m['last'], **packed)
        cm.dot_gated(m['w2'].T, m['s'], m['b2'], target=m['y'], pre=m['halves'])
        m['y'].add(m['x'])
        cm.dot(m['e'].T, m['y'], target=m['logits'])
        cm.log_probs(m['logits'], m['aims'], logp=m['logp'], log_z=m['log_z'])
        dl = cm.log_probs_grad(m['logits'], m['aims'], m['log_z'], m['lw'])
        cm.dot(m['y'], dl.T, target=m['de'])
        cm.dot(m['e'], dl, target=m['dy'])
        cm.dot_gated_grad(m['dy'], m['w2'].T, m['s'], m['halves'], m1_grad=m['dw2'], m2_grad=m['ds'], bias_grad=m['db2'])
        cm.gated_scan_grad(m['ds'], m['pre'], m['s'], state_grad=m['dstate'], **packed)             # over pre
        cm.dot(m['h'], m['pre'].T, target=m['dw1'])
        cm.dot(m['w1'], m['pre'], target=m['dh'])
        cm.layer_norm_grad(m['dh'], m['x'], m['g'], target=m['dx'], gain_grad=m['dg'], bias_grad=m['dc'])
        m['dx'].add(m['dy'])
        cm.embed_grad(m['dx'], m['labels'], m['de'], mult=2.0, beta=1.0)                            # the table's second use

    def oracle(self, h):
        x = seq.embed(h['e'], h['labels'], 2.0)
        n = tok.layer_norm(x, h['g'], h['c'])
        pre = h['w1'].T @ n
        s = np.nan_to_num(seq.gated_scan(pre, self.at, h['state'])[0])
        y, halves = tok.dot_gated(h['w2'].T, s, h['b2'])
        y = y + x
        logits = h['e'].T @ y
        o = tok.log_probs(logits, h['aims'])
        dl = tok.log_probs_grad(logits, h['aims'], o['log_z'], h['lw'])
        g, dy = dict(), h['e'] @ dl
        dp = tok.gate_grad(dy, halves)
        g['dw2'], g['db2'] = s @ dp.T, dp.sum(axis=1, keepdims=True)
        dpre, g['dstate'] = seq.gated_scan_grad(h['w2'] @ dp, pre, s, self.at, h['state'])[:2]
        dpre = np.nan_to_num(dpre)
        g['dw1'] = n @ dpre.T
        dx, g['dg'], g['dc'] = tok.layer_norm_grad(h['w1'] @ dpre, x, h['g'])
        g['de'] = y @ dl.T + seq.embed_grad(dx + dy, h['labels'], h['e'].shape[1], 2.0)[0]
        return float((h['lw'] * o['logp']).sum()), g, o


def test_a_net_over_packed_texts_forward_and_backward(cm, rng):
    """All of them as they are used.  Every gradient against the oracle's (a chain of ten operators, each off by 10 u to 100 u of the magnitudes that
    it handles: 2e-5 of the largest entry), and along random directions against differences of the oracle's objective."""
    b = Net(cm, rng)
    b.m['pre'].assign(0.0)                                                # (columns behind the last text stay: no gradient comes from them)
    b.step()
    pad = slice(b.at[-1], b.w)
    value, grads, o = b.oracle(b.host)
    assert np.max(np.abs(b.m['logp'].asarray() - o['logp'])) < 1e-5 * np.max(np.abs(o['logp']))
    assert not b.m['dy'].asarray()[:, pad].any()
    for name in b.GRADS:
        got, want = b.m[name].asarray(), grads[name]
        if name == 'dw1':                                                 # (behind the last text the derivative of pre is what was there: pre itself)
            n = tok.layer_norm(seq.embed(b.host['e'], b.host['labels'], 2.0), b.host['g'], b.host['c'])[:, pad]
            want = want + n @ (b.host['w1'].T @ n).T
        if name in ('dg', 'dc', 'de'):
            continue
        assert np.max(np.abs(got - want)) < 2e-5 * np.max(np.abs(want)), name
    # the same without padding: every gradient
    b = Net(cm, rng, pad=0)
    b.step()
    value, grads, o = b.oracle(b.host)
    for name in b.GRADS:
        got, want = b.m[name].asarray(), grads[name]
        assert np.max(np.abs(got - want)) < 2e-5 * np.max(np.abs(want)), name
        way = rng.standard_normal(want.shape)
        ends = []
        for s in (1e-5, -1e-5):
            h = dict(b.host)
            h[name[1:]] = h[name[1:]] + s * way
            ends.append(b.oracle(h)[0])
        slope = (ends[0] - ends[1]) / 2e-5
        assert abs(np.sum(got * way) - slope) < 1e-4 * np.max(np.abs(want)) * np.sqrt(want.size) + 1e-6 * (1 + abs(value)), name


class ZerosBehind(object):
    """The library, but that the derivative by the gates and inputs goes into a matrix of zeros first, for products that take the padding too."""

    def __init__(self, cm, shape):
        self.cm, self.zeros = cm, cm.CUDAMatrix(F(np.zeros(shape)))

    def __getattr__(self, name):
        return getattr(self.cm, name)

    def gated_scan_grad(self, deriv, pre, out, **args):
        pre.assign(self.cm.gated_scan_grad(deriv, pre, out, target=self.zeros, **args))


def test_a_net_over_packed_and_padded_texts(cm, rng):
    """Every gradient, with padding behind the last text; bounds as above."""
    b = Net(cm, rng)
    b.cm = ZerosBehind(cm, b.m['pre'].shape)
    for _ in range(2):
        b.step()
        value, grads, o = b.oracle(b.host)
        for name in b.GRADS:
            got, want = b.m[name].asarray(), grads[name]
            assert np.max(np.abs(got - want)) < 2e-5 * np.max(np.abs(want)), name


def test_recorded_nets_and_eager_calls_between_them(cm):
    """Two recordings of different sizes that share the library's workspaces, replayed in turn with eager calls of a third size between them."""
    sizes = (dict(), dict(d=200, f=130, v=3000, at=(0, 700, 1500), pad=0), dict(d=33, f=20, v=100, at=(0, 5, 3000), pad=3))
    nets = [Net(cm, np.random.default_rng(i), **s) for i, s in enumerate(sizes)]
    names = Net.GRADS + ('logp', 'last', 's')
    want = []
    for b in nets:
        for _ in range(2):
            b.step()
        want.append(bits(b.m[n] for n in names))
    graphs = []
    for b in nets[:2]:
        with cm.Graph() as g:
            b.step()
        graphs.append(g)
    for i in range(4):
        for b, g, w in zip(nets, graphs, want):
            for n in names:
                if n != 's':
                    b.m[n].assign(-3.0)
            nets[2].step()
            g.launch()
            nets[2].step()
            assert all(np.array_equal(p, q) for p, q in zip(bits(b.m[n] for n in names), w)), i
            assert all(np.array_equal(p, q) for p, q in zip(bits(nets[2].m[n] for n in names), want[2])), i


class Decoder(object):
    """One step of answering: the drawn tokens' columns, a recurrence from state to state, logits, the next tokens; all on the device."""

    def __init__(self, cm, rng, d=40, f=64, v=700, n=5):
        D = lambda *s: cm.CUDAMatrix(F(rng.standard_normal(s)))
        self.cm, self.e, self.w1, self.w2, self.state = cm, D(d, v), D(d, 2 * f), D(f, v), D(f, n)
        self.tokens, self.uniform, self.logp = cm.CUDAMatrix(F([[0.0] * n])), cm.empty((1, n)), cm.empty((1, n))
        self.x, self.pre, self.h, self.logits = cm.empty((d, n)), cm.empty((2 * f, n)), cm.empty((f, n)), cm.empty((v, n))

    def step(self):
        cm = self.cm
        cm.embed(self.e, self.tokens, target=self.x, mult=0.3)
        cm.dot(self.w1.T, self.x, target=self.pre)
        cm.gated_scan(self.pre, target=self.h, state=self.state, last=self.state)
        cm.dot(self.w2.T, self.h, target=self.logits)
        self.uniform.fill_with_rand()
        cm.sample_tokens(self.logits, self.uniform, target=self.tokens, temperature=0.8, top_k=40, top_p=0.9, logp=self.logp)


def test_recorded_decoding_is_the_eager_one(cm):
    a, b = Decoder(cm, np.random.default_rng(3)), Decoder(cm, np.random.default_rng(3))
    cm.CUDAMatrix.init_random(7)
    want = []
    for _ in range(12):
        a.step()
        want.append((a.tokens.asarray().copy(), a.logp.asarray().copy(), a.state.asarray().copy()))
        logits, u = a.logits.asarray(), a.uniform.asarray()[0]
        for c in range(logits.shape[1]):
            assert want[-1][0][0, c] == seq.sample_token(logits[:, c], u[c], temperature=0.8, top_k=40, top_p=0.9)[0]
    cm.CUDAMatrix.init_random(7)
    got = []
    def keep():
        got.append((b.tokens.asarray().copy(), b.logp.asarray().copy(), b.state.asarray().copy()))
    b.step()
    keep()
    with cm.Graph() as g:
        b.step()
    for _ in range(11):
        g.launch()
        keep()
    assert all(np.array_equal(p, q) for x, y in zip(got, want) for p, q in zip(x, y))
    cm.CUDAMatrix.init_random(1)


def test_a_net_on_a_stream_of_the_callers(cm):
    hip = ct.CDLL('libamdhip64.so')
    a, b = Net(cm, np.random.default_rng(9), pad=0), Net(cm, np.random.default_rng(9), pad=0)
    a.step()
    want = bits(a.m[n] for n in Net.GRADS)
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
    assert all(np.array_equal(p, q) for p, q in zip(bits(b.m[n] for n in Net.GRADS), want))
    assert hip.hipStreamDestroy(stream) == 0
