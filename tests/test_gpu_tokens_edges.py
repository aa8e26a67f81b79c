"""Ends of the ranges of the operators on columns of tokens.  Bounds and helpers of test_gpu_tokens.py."""
import ctypes as ct

import numpy as np
import pytest

from oracle import token_oracle as tok
from test_gpu_tokens import F, U, act_bounds, bits, check, check_log_probs, device, gated_check, grad_bounds, neighbours_untouched, norm_bound

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------ top lists

@pytest.mark.parametrize("h,w", [(1025, 40), (4096, 40), (5000, 40), (32000, 600), (131072, 2), (200001, 10)])
@pytest.mark.parametrize("lowest", [-1e9, float(np.finfo(np.float32).min), -np.inf])
def test_log_probs_of_a_mask_that_leaves_one_entry_fewer_than_asked_for(cm, h, w, lowest):
    """k - 1 entries are allowed, in as many lanes or in few, row 0 masked or not: the last of the list is the first masked row.  What
    is left unwritten stays NaN."""
    rng = np.random.default_rng(h + w)
    labels = F(rng.integers(0, h, (1, w)))
    for k in (2, 5, 20, 64):
        x = F(np.full((h, w), lowest))
        few = range(w) if w < 100 else list(range(24)) + list(range(w - 8, w))           # (columns that the oracle looks at)
        for c in range(w):
            n = k - 1 if c % 4 < 3 else int(rng.integers(0, k))
            step = 4 if c % 2 else 1                                  # (every row of a lane's group, or other groups)
            rows = 1 + step * rng.choice((h - 1) // step, n, replace=False)
            if c % 8 == 5 and n:
                rows[0] = 0
            x[rows, c] = rng.standard_normal(n)
        names = dict(logp=(1, w), entropy=(1, w), log_z=(1, w), top=(k, w), top_labels=(k, w))
        out = {name: cm.CUDAMatrix(F(np.full(shape, np.nan))) for name, shape in names.items()}
        cm.log_probs(cm.CUDAMatrix(x), cm.CUDAMatrix(labels), **out)
        few = list(few)
        got = {name: m.asarray()[:, few] for name, m in out.items()}
        assert not np.isnan(out['top_labels'].asarray()).any(), (h, w, k)
        check_log_probs(x[:, few], labels[:, few], k, got)


# ------------------------------------------------------------------ more columns than one launch takes

def ends(mat, n):
    """The first, and the last n columns, where a call of more than one launch joins, and those around the middle."""
    w = mat.shape[1]
    return [mat.slice(a, a + n).asarray().copy() for a in (0, (w - n) // 2, w - n)]


def wide(cm, rng, h, w, n):
    """h x w with random columns at the places of `ends`, and those (the rest is constant)."""
    big = cm.empty((h, w))
    big.assign(0.125)
    parts = [F(rng.standard_normal((h, n))) for _ in range(3)]
    for a, p in zip((0, (w - n) // 2, w - n), parts):
        src = cm.CUDAMatrix(p)
        big.slice(a, a + n).assign(src)
        src.free_device_memory()
    return big, parts


def release(*mats):
    for m in mats:
        m.free_device_memory()


@pytest.mark.parametrize("h,w,k", [(1, (1 << 24) + 5, 1), (2, (1 << 24) + 3, 0), (3, (1 << 25) + 7, 2), (4, (1 << 26) + 5, 1), (10, (1 << 26) + 5, 0)])
def test_log_probs_of_more_columns_than_a_launch_takes(cm, rng, h, w, k):
    n = 40
    big, parts = wide(cm, rng, h, w, n)
    labels = cm.empty((1, w))
    labels.assign(float(h - 1))
    out = {name: cm.empty((1, w)) for name in ('logp', 'entropy', 'log_z')}
    if k:
        out.update(top=cm.empty((k, w)), top_labels=cm.empty((k, w)))
    for m in out.values():
        m.assign(np.nan)
    cm.log_probs(big, labels, **out)
    got = {name: ends(m, n) for name, m in out.items()}
    for i, p in enumerate(parts):
        check_log_probs(p, F(np.full((1, n), h - 1)), k, {name: g[i] for name, g in got.items()})
    # every column of the rest has the same result, and has been written
    rest = out['log_z'].slice(n, (w - n) // 2).asarray()
    assert (rest == rest[0, 0]).all() and abs(rest[0, 0] - (0.125 + np.log(h))) < 1e-6
    release(big, labels, *out.values())


@pytest.mark.parametrize("h,w", [(1, (1 << 26) + 5), (7, (1 << 26) + 33), (1025, (1 << 24) + 9)])
def test_log_probs_grad_of_more_columns_than_a_launch_takes(cm, rng, h, w):
    """In place.  Bound: log p is off by 2 u |log p| (x - log_z, and what exp2 takes), p by that and 3 u of it; every product and sum adds u of
    its terms, the entropy term has log p twice."""
    n = 40
    big, parts = wide(cm, rng, h, w, n)
    rows = dict(labels=h - 1.0, log_z=1.0 + np.log(h), logp_weight=-0.75, entropy=0.5, entropy_weight=0.25)
    M = {}
    for name, v in rows.items():
        M[name] = cm.empty((1, w))
        M[name].assign(v)
    cm.log_probs_grad(big, M['labels'], M['log_z'], M['logp_weight'], M['entropy'], M['entropy_weight'])
    row = {name: np.full((1, n), np.float32(v)) for name, v in rows.items()}
    for p, got in zip(parts, ends(big, n)):
        want = tok.log_probs_grad(p, row['labels'], row['log_z'], row['logp_weight'], row['entropy'], row['entropy_weight'])
        lp = p.astype(np.float64) - row['log_z']
        perr = np.exp(lp) * (2 * np.abs(lp) + 3)
        check(got, want, U * (0.75 * (perr + 2 + 2 * np.exp(lp)) + 0.25 * (perr * (np.abs(lp) + 0.5) + np.exp(lp) * (2 * np.abs(lp) + 1)) + 2 * np.abs(want)))
    rest = big.slice(n, n + 1000).asarray()
    assert (big.slice((w + n) // 2, (w + n) // 2 + 1000).asarray() == rest[:, :1]).all() and (rest != 0.125).all()
    release(big, *M.values())


def test_elementwise_calls_of_more_entries_than_a_launch_takes(cm):
    """2^34 entries and some, four a lane: all of them are written."""
    h, w = 1 << 17, (1 << 17) + 3
    big = cm.empty((h, w))
    big.assign(0.0)
    big.assign(-1.5)
    for c in (0, 1, w // 2, (1 << 17) - 1, 1 << 17, w - 1):
        assert (big.slice(c, c + 1).asarray() == -1.5).all(), c
    big.add(2.0)
    for c in (0, 1, w // 2, (1 << 17) - 1, 1 << 17, w - 1):
        assert (big.slice(c, c + 1).asarray() == 0.5).all(), c
    release(big)


@pytest.mark.parametrize("skip,h,w", [(1, 1 << 16, (1 << 16) + 3), (0, 1 << 17, (1 << 17) + 3)])
def test_copies_of_more_entries_than_a_launch_takes(cm, skip, h, w):
    """From an address off 16 bytes an entry a lane, 2^32 of them and some; else four a lane."""
    whole = cm.empty((h, w + 1))
    whole.assign(2.5)
    mat = cm.cudamat()
    ct.memmove(ct.pointer(mat), whole.p_mat, ct.sizeof(mat))
    mat.data_device = ct.cast(ct.addressof(mat.data_device.contents) + 4 * skip, type(mat.data_device))
    mat.owns_data, mat.size[1] = 0, w
    src = cm.CUDAMatrix(mat)
    dst = cm.empty((h, w))
    dst.assign(0.0)
    dst.assign(src)
    for c in (0, 1, w // 2, h - 1, h, w - 1):
        assert (dst.slice(c, c + 1).asarray() == 2.5).all(), c
    release(dst, whole)


def test_a_call_without_a_launch_is_an_error_and_the_next_one_is_none(cm):
    """normlimit takes four columns a workgroup in one launch: 2^26 of them are refused and left as they are."""
    wide_one, row = cm.empty((4, 1 << 26)), cm.empty((4, 1000))
    wide_one.assign(3.0)
    row.assign(3.0)
    with pytest.raises(cm.CUDAMatException):
        wide_one.norm_limit(1.0, axis=0)
    assert (wide_one.slice(0, 1000).asarray() == 3.0).all() and (wide_one.slice((1 << 26) - 1000, 1 << 26).asarray() == 3.0).all()
    row.norm_limit(1.0, axis=0)
    assert np.allclose(row.asarray(), 0.5, rtol=1e-6)
    release(wide_one, row)


@pytest.mark.parametrize("f,w,acts", [(1, (1 << 26) + 5, ('silu',)), (3, (1 << 26) + 7, ('relu',))])
def test_the_halves_of_more_columns_than_a_launch_takes(cm, rng, f, w, acts):
    """The pass over the halves, backward, in the place of pre."""
    n = 40
    for act in acts:
        dy, dys = wide(cm, rng, f, w, n)
        pre, pres = wide(cm, rng, 2 * f, w, n)
        m1, m2 = cm.empty((2 * f, 1)), cm.empty((1, w))                     # (their values are not read: no gradient of theirs is asked for)
        assert cm.dot_gated_grad(dy, m1, m2, pre, act=act) is pre
        for d, p, got in zip(dys, pres, ends(pre, n)):
            want = tok.gate_grad(d, p, act)
            ve, se = act_bounds(act, p[:f].astype(np.float64), 0.0)
            ad, au = np.abs(d.astype(np.float64)), np.abs(p[f:].astype(np.float64))
            check(got, want, np.vstack([ad * au * se, ad * ve]) + 4 * U * np.abs(want))
        rest = pre.slice(n, n + 500).asarray()
        assert (pre.slice((w + n) // 2, (w + n) // 2 + 500).asarray() == rest[:, :1]).all() and (rest != 0.125).all()
        release(dy, pre, m1, m2)


def test_dot_gated_of_more_units_than_a_launch_takes(cm, rng):
    """One column and one term: products of two numbers."""
    f, n = (1 << 26) + 5, 40
    w, parts = wide(cm, rng, 1, 2 * f, n)
    gate, up = w.slice(0, n).asarray().copy(), w.slice(2 * f - n, 2 * f).asarray().copy()
    x, y = cm.CUDAMatrix(F([[1.5]])), cm.empty((f, 1))
    y.assign(np.nan)
    cm.dot_gated(w.T, x, target=y, act='relu')
    y.reshape((1, f))
    at = w.slice(f, f + n).asarray().astype(np.float64)
    got, last = y.slice(0, n).asarray(), y.slice(f - n, f).asarray()
    check(got, np.maximum(1.5 * gate, 0) * 1.5 * at, 4 * U * np.abs(2.25 * gate * at))
    g = 1.5 * w.slice(f - n, f).asarray().astype(np.float64)
    check(last, np.maximum(g, 0) * 1.5 * up, 4 * U * np.abs(g * 1.5 * up))
    assert not np.isnan(y.asarray()).any()
    release(w, x, y)


def test_counter_dropout_of_more_entries_than_a_launch_takes(cm, rng):
    """2^34 entries and some, in place: counters go on past 2^32."""
    h, w, n = 1 << 17, (1 << 17) + 3, 2
    big, parts = wide(cm, rng, h, w, n)
    cm.counter_dropout(big, 0.25, 77, stream=5, mult=2.0)
    for a, p, got in zip((0, (w - n) // 2, w - n), parts, ends(big, n)):
        keep = tok.dropout_keep((h, n), 0.25, 77, stream=5, first=h * a, count=h * n).reshape((h, n), order='F')
        assert np.array_equal(got, np.where(keep, 2 * p, np.float32(0))), a
    for c in ((1 << 17) - 2, (1 << 17) - 1, 1 << 17):                   # (where the second launch begins)
        keep = tok.dropout_keep((h, 1), 0.25, 77, stream=5, first=h * c, count=h).reshape((h, 1))
        assert np.array_equal(big.slice(c, c + 1).asarray(), np.where(keep, np.float32(0.25), np.float32(0))) or c >= w - n, c
    release(big)


@pytest.mark.parametrize("h", [3, 4])
def test_layer_norm_of_more_columns_than_a_launch_takes(cm, rng, h):
    """2^29 columns and some, forward and backward in place; constant columns give the bias, and add nothing to the gain's gradient."""
    w, n = (1 << 29) + 37, 40
    big, parts = wide(cm, rng, h, w, n)
    gain, bias = F(1 + 0.3 * rng.standard_normal((h, 1))), F(rng.standard_normal((h, 1)))
    G, B = cm.CUDAMatrix(gain), cm.CUDAMatrix(bias)
    cm.layer_norm(big, G, B)
    for p, got in zip(parts, ends(big, n)):
        want = tok.layer_norm(p, gain, bias)
        check(got, want, norm_bound(p, gain, want))
    for c in (n, (1 << 29) - 500, w // 2 + n):
        assert (big.slice(c, c + 400).asarray() == bias).all(), c
    release(big)
    x, xs = wide(cm, rng, h, w, n)
    dy, dys = wide(cm, rng, h, w, n)
    gg, gb = cm.empty((h, 1)), cm.empty((h, 1))
    gg.assign(2.0)
    gb.assign(2.0)
    cm.layer_norm_grad(dy, x, G, gain_grad=gg, bias_grad=gb, mult=0.5, beta=3.0)
    wg, wb, eg, eb = 6.0, 6.0 + 0.5 * 0.125 * (w - 3 * n), 0.0, 0.125 * (w - 3 * n)
    for p, d, got in zip(xs, dys, ends(dy, n)):
        dx, dg, db = tok.layer_norm_grad(d, p, gain)
        ex, e1, e2 = grad_bounds(d, p, gain)
        check(got, dx, ex)
        wg, wb, eg, eb = wg + 0.5 * dg, wb + 0.5 * db, eg + e1, eb + np.abs(d.astype(np.float64)).sum(axis=1, keepdims=True)
    # (a lane adds up every 16384th column or fewer)
    check(gg.asarray(), wg, 0.5 * eg + 4 * U * (np.abs(wg) + 6))
    check(gb.asarray(), wb, U * (w / 16384 + 100) * 0.5 * eb + 4 * U * (np.abs(wb) + 6))
    release(x, dy, gg, gb, G, B)


# ------------------------------------------------------------------ tall columns

@pytest.mark.parametrize("h", [16390, 20000, 100000, 1000003])
def test_layer_norm_of_tall_columns_far_from_zero(cm, h):
    """Columns that are constant give the bias, whatever their value (the sum of equal entries is exact in 64 bits, and so is its quotient by
    their number): nothing is NaN.  Entries that differ by a few steps of fp32: the mean is taken as m + d with |d| of half a step of m, so the
    variance is off by chain u of itself and d^2, which is no more than twice it here."""
    rng = np.random.default_rng(h)
    values = [3.0, 98765.4, -1000000.3, 7.7e7, 1e9, 3e38, -1e-30]
    x = F(np.repeat(F([values]), h, axis=0))
    steps = F(98765.4 + 2.0 ** -7 * rng.integers(-2, 3, (h, 1)))
    dy, gain, bias = F(rng.standard_normal((h, 8))), F(1 + 0.3 * rng.standard_normal((h, 1))), F(rng.standard_normal((h, 1)))
    x = F(np.hstack([x, steps]))
    y = cm.layer_norm(cm.CUDAMatrix(x), cm.CUDAMatrix(gain), cm.CUDAMatrix(bias), target=cm.empty(x.shape)).asarray()
    assert np.array_equal(y[:, :7], np.repeat(bias, 7, axis=1))
    want = tok.layer_norm(x[:, 7:], gain, bias)
    check(y[:, 7:], want, 3 * norm_bound(x[:, 7:], gain, want))
    G, dx, gg, gb = cm.CUDAMatrix(gain), cm.empty(x.shape), cm.empty((h, 1)), cm.empty((h, 1))
    cm.layer_norm_grad(cm.CUDAMatrix(dy), cm.CUDAMatrix(x), G, target=dx, gain_grad=gg, bias_grad=gb)
    want, wg, wb = tok.layer_norm_grad(dy, np.hstack([np.repeat(F([[3.0]]), 7, axis=1) * np.ones((h, 1)), x[:, 7:]]), gain)
    ex, eg, eb = grad_bounds(dy, F(np.hstack([np.full((h, 7), 3.0), x[:, 7:]])), gain)
    check(dx.asarray(), want, 3 * ex)
    check(gg.asarray(), wg, 3 * eg)
    check(gb.asarray(), wb, eb)


# ------------------------------------------------------------------ what else is queued

@pytest.mark.parametrize("m,n,k", [(500, 100, 100), (256, 256, 64), (300, 200, 120), (1000, 64, 128)])
def test_a_product_that_waits_keeps_its_kernel_beside_a_gated_gradient(cm, rng, m, n, k):
    """dot may hold its launch back until the next call; the gradient's own choice of tiles (64 columns, no units: nothing but the fill of
    m2_grad is launched) is not for it."""
    a, b = cm.CUDAMatrix(F(rng.standard_normal((k, m)))), cm.CUDAMatrix(F(rng.standard_normal((k, n))))
    want, got = cm.empty((m, n)), cm.empty((m, n))
    cm.dot(a.T, b, target=want)
    want = want.asarray().copy()
    w, x, dx, dy, pre = cm.empty((7, 0)), cm.empty((7, 64)), cm.empty((7, 64)), cm.empty((0, 64)), cm.empty((0, 64))
    dx.assign(5.0)
    wt, at = w.T, a.T
    cm.cuda_sync_threads()
    cm.dot(at, b, target=got)
    cm.dot_gated_grad(dy, wt, x, pre, m2_grad=dx)
    assert np.array_equal(got.asarray(), want) and not dx.asarray().any()


# ------------------------------------------------------------------ offsets beyond 2^31 entries, at ordinary heights

@pytest.mark.parametrize("h", [64, 1023, 2050])
def test_columns_beyond_two_to_the_31_entries(cm, rng, h):
    """The kernels that hold columns in registers (16 lanes, a wavefront, a workgroup), in place: the last columns against the definitions."""
    w, n = (1 << 31) // h + 200, 40
    gain, bias = F(1 + 0.3 * rng.standard_normal((h, 1))), F(rng.standard_normal((h, 1)))
    G, B = cm.CUDAMatrix(gain), cm.CUDAMatrix(bias)
    big, parts = wide(cm, rng, h, w, n)
    cm.layer_norm(big, G, B)
    for p, got in zip(parts, ends(big, n)):
        want = tok.layer_norm(p, gain, bias)
        check(got, want, norm_bound(p, gain, want))
    release(big)
    x, xs = wide(cm, rng, h, w, n)
    labels, rows = cm.empty((1, w)), {name: cm.empty((1, w)) for name in ('logp', 'entropy', 'log_z')}
    labels.assign(h - 3.0)
    cm.log_probs(x, labels, **rows)
    got = {name: ends(m, n) for name, m in rows.items()}
    for i, p in enumerate(xs):
        check_log_probs(p, F(np.full((1, n), h - 3)), 0, {name: g[i] for name, g in got.items()})
    dy, dys = wide(cm, rng, h, w, n)
    gg, gb = cm.empty((h, 1)), cm.empty((h, 1))
    cm.layer_norm_grad(dy, x, G, gain_grad=gg, bias_grad=gb)
    wg, eg = 0.0, 0.0
    for p, d, got in zip(xs, dys, ends(dy, n)):
        dx, dg, _ = tok.layer_norm_grad(d, p, gain)
        ex, e1, _ = grad_bounds(d, p, gain)
        check(got, dx, ex)
        wg, eg = wg + dg, eg + e1
    check(gg.asarray(), wg, eg + 4 * U * np.abs(wg))                    # (constant columns of 0.125 add nothing)
    lw = F(np.full((1, n), -1.0))
    ones = cm.empty((1, w))
    ones.assign(-1.0)
    log_z = [z.astype(np.float64) for z in ends(rows['log_z'], n)]
    cm.log_probs_grad(x, labels, rows['log_z'], ones)
    for p, z, got in zip(xs, log_z, ends(x, n)):
        want = tok.log_probs_grad(p, np.full((1, n), h - 3.0), z, lw)
        lp = p.astype(np.float64) - z
        check(got, want, U * (np.exp(lp) * (2 * np.abs(lp) + 4) + 2 * np.abs(want) + np.exp(lp)))
    release(x, dy, labels, ones, gg, gb, G, B, *rows.values())


def test_halves_and_results_beyond_two_to_the_31_entries(cm, rng):
    """pre of 2 f rows passes 2^31 entries at half the columns: the pass over the halves, and the stores of a gated product on tiles."""
    f, n = 1000, 40
    w = (1 << 31) // (2 * f) + 200
    dy, dys = wide(cm, rng, f, w, n)
    pre, pres = wide(cm, rng, 2 * f, w, n)
    m1, m2 = cm.empty((2 * f, 1)), cm.empty((1, w))
    cm.dot_gated_grad(dy, m1, m2, pre, act='relu')
    for d, p, got in zip(dys, pres, ends(pre, n)):
        want = tok.gate_grad(d, p, 'relu')
        check(got, want, 4 * U * np.abs(want))
    release(dy, m1, m2)
    d = 32
    wt = F(rng.standard_normal((d, 2 * f)) / np.sqrt(d))
    x, xs = wide(cm, rng, d, w, n)
    y = cm.empty((f, w))
    cm.dot_gated(cm.CUDAMatrix(wt).T, x, target=y, pre=pre, act='silu')
    for p, got, halves in zip(xs, ends(y, n), ends(pre, n)):
        gated_check(cm, wt, p, None, 'silu', got, halves)
    release(x, y, pre)


# ------------------------------------------------------------------ operands stored either way, anywhere

@pytest.mark.parametrize("d,f,n", [(70, 33, 1), (70, 33, 9), (257, 130, 20), (64, 100, 65), (130, 70, 300), (256, 256, 256)])
@pytest.mark.parametrize("skip", [0, 1, 3])
def test_dot_gated_grad_of_operands_stored_either_way_with_sums(cm, rng, d, f, n, skip):
    """Weights and inputs stored either way, every operand and result off a 16-byte boundary, the gradients accumulated and scaled, that of the
    bias among them.  The halves' derivatives are read back, so the bounds are those of the products and sums."""
    w, x, dy = F(rng.standard_normal((d, 2 * f)) / np.sqrt(d)), F(rng.standard_normal((d, n))), F(rng.standard_normal((f, n)))
    pre, old = F(rng.standard_normal((2 * f, n))), F(rng.standard_normal((d, 2 * f)))
    aw, ax = np.abs(w.astype(np.float64)), np.abs(x.astype(np.float64))
    for wt in (False, True):
        for xt in (False, True):
            W, X = device(cm, w if wt else w.T, skip), device(cm, x.T if xt else x, skip)
            dw, dx, db = device(cm, old if wt else old.T, skip), device(cm, np.full(X.shape, np.nan), skip), device(cm, np.full((2 * f, 1), 2.0), skip)
            t = device(cm, np.zeros((2 * f, n)), skip)
            cm.dot_gated_grad(device(cm, dy, skip), W.T if wt else W, X.T if xt else X, device(cm, pre, skip), target=t, m1_grad=dw, m2_grad=dx,
                              bias_grad=db, mult=-0.5, beta=0.25)
            got = t.asarray().astype(np.float64)
            ve, se = act_bounds('silu', pre[:f].astype(np.float64), 0.0)
            ad, au = np.abs(dy.astype(np.float64)), np.abs(pre[f:].astype(np.float64))
            check(got, tok.gate_grad(dy, pre, 'silu'), np.vstack([ad * au * se, ad * ve]) + 4 * U * np.abs(got), ('halves', wt, xt))
            at, c = np.abs(got), U * (n / 4 + 24)
            wdw, wdx, wdb = x.astype(np.float64) @ got.T, w.astype(np.float64) @ got, got.sum(axis=1, keepdims=True)
            want = 0.25 * old - 0.5 * wdw
            check(dw.asarray() if wt else dw.asarray().T, want, 0.5 * c * (ax @ at.T) + 3 * U * (0.25 * np.abs(old) + np.abs(wdw)), ('weights', wt, xt))
            check(dx.asarray().T if xt else dx.asarray(), wdx, U * (f / 2 + 24) * (aw @ at), ('inputs', wt, xt))
            check(db.asarray(), 0.5 - 0.5 * wdb, 0.5 * c * at.sum(axis=1, keepdims=True) + 3 * U * (0.5 + np.abs(wdb)), ('bias', wt, xt))
            for m in (W, X, dw, dx, db, t):
                neighbours_untouched(m, skip)


def test_an_infinite_column_of_a_gated_product_is_in_all_of_its_results(cm, rng):
    """Sigmoid gates: 0 or 1 times an infinity, or 0 times one (NaN); no result of that column is finite."""
    for d, f, n in ((64, 40, 6), (300, 700, 300), (1024, 1500, 1500), (64, 40, 11), (2048, 30, 6), (100, 60, 16), (512, 2050, 40)):
        w, x = F(rng.standard_normal((d, 2 * f)) / np.sqrt(d)), F(rng.standard_normal((d, n)))
        x[5, 4] = np.inf
        y = cm.dot_gated(cm.CUDAMatrix(w).T, cm.CUDAMatrix(x), act='sigmoid').asarray()
        ok = w[5, :f] > 0                                   # (a gate of 0 leaves the sign of 0 times infinity: NaN; one of 1 the infinity)
        want = np.where(ok, np.where(w[5, f:] > 0, np.inf, -np.inf), np.nan)
        assert not np.isfinite(y[:, 4]).any() and np.array_equal(y[:, 4], want, equal_nan=True), (d, f, n)
        cols = [c for c in range(n) if c != 4]
        gated_check(cm, w, x[:, cols], None, 'sigmoid', y[:, cols], None)


# ------------------------------------------------------------------ lists of anything

def any_column(rng, h):
    """Entries with ties, masks of one kind or several, NaN and infinities in places of any number."""
    kind = rng.integers(7)
    x = rng.standard_normal(h)
    if kind == 1:
        x = np.round(x)
    elif kind >= 2:
        x = np.full(h, rng.choice([-1e9, np.finfo(np.float32).min, -np.inf, 0.0, -0.0]))
        at = rng.choice(h, min(h, int(rng.choice([0, 1, 3, 4, 5, 19, 20, 63, 64, 65, 300]))), replace=False)
        x[at] = 2.0 if kind == 3 else rng.standard_normal(at.size)
        if kind == 4:
            x[rng.integers(0, h, 30)] = np.nan
        elif kind == 5:
            a, b = np.sort(rng.integers(0, h + 1, 2))
            x[a:b] = -np.inf
        elif kind == 6:
            x[rng.integers(0, h, 3)] = rng.choice([np.inf, 0.0, -0.0])
    return x


@pytest.mark.parametrize("h,w", [(4, 64), (37, 64), (257, 64), (1000, 64), (1024, 64), (1025, 64), (1027, 64), (4095, 64), (4099, 64), (9001, 64), (9001, 600), (30000, 40), (70003, 9)])
@pytest.mark.parametrize("k", [1, 2, 4, 5, 20, 63, 64])
def test_lists_of_any_columns(cm, h, w, k):
    k = min(k, h)
    rng = np.random.default_rng(100 * h + k)
    few = min(w, 64)
    x = F(np.stack([any_column(rng, h) for _ in range(few)], axis=1))
    if w > few:
        x = F(np.tile(x, (1, w // few + 1))[:, :w])
    labels = F(rng.integers(-1, h, (1, w)))
    names = dict(logp=(1, w), entropy=(1, w), log_z=(1, w), top=(k, w), top_labels=(k, w))
    out = {name: cm.CUDAMatrix(F(np.full(shape, 7.0))) for name, shape in names.items()}
    cm.log_probs(cm.CUDAMatrix(x), cm.CUDAMatrix(labels), **out)
    check_log_probs(x[:, -few:], labels[:, -few:], k, {name: m.asarray()[:, -few:] for name, m in out.items()})


# ------------------------------------------------------------------ recordings that share workspaces

def test_two_recordings_of_calls_with_workspaces(cm, rng):
    """Columns in segments, sums of several workgroups, gradients of few and of many columns: two graphs of different sizes, replayed in turn
    with eager calls of a third size between them, each with the bits of the calls by themselves."""
    class Set(object):
        def __init__(self, v, c, d, f, n):
            D = lambda *s: cm.CUDAMatrix(F(rng.standard_normal(s)))
            self.x, self.labels, self.top = D(v, c), cm.CUDAMatrix(F(rng.integers(0, v, (1, c)))), 5
            self.rows, self.lists = [cm.empty((1, c)) for _ in range(3)], [cm.empty((5, c)) for _ in range(2)]
            self.dy, self.h, self.g = D(d, 700), D(d, 700), D(d, 1)
            self.dh, self.gg, self.gb = cm.empty((d, 700)), cm.empty((d, 1)), cm.empty((d, 1))
            self.w, self.in_, self.dg, self.pre = D(d, 2 * f), D(d, n), D(f, n), D(2 * f, n)
            self.t, self.dw, self.dx, self.db, self.y = cm.empty((2 * f, n)), cm.empty((d, 2 * f)), cm.empty((d, n)), cm.empty((2 * f, 1)), cm.empty((f, n))

        def step(self):
            cm.log_probs(self.x, self.labels, *(self.rows + self.lists))
            cm.layer_norm_grad(self.dy, self.h, self.g, target=self.dh, gain_grad=self.gg, bias_grad=self.gb)
            cm.dot_gated(self.w.T, self.in_, target=self.y)
            cm.dot_gated_grad(self.dg, self.w.T, self.in_, self.pre, target=self.t, m1_grad=self.dw, m2_grad=self.dx, bias_grad=self.db)

        def out(self):
            return self.rows + self.lists + [self.dh, self.gg, self.gb, self.t, self.dw, self.dx, self.db, self.y]

    a, b, c = Set(50001, 3, 300, 200, 5), Set(20000, 17, 130, 40, 3), Set(100000, 2, 64, 700, 14)
    want = []
    for s in (a, b, c):
        s.step()
        want.append(bits(s.out()))
    graphs = []
    for s in (a, b):
        with cm.Graph() as g:
            s.step()
        graphs.append(g)
    for i in range(4):
        for s, g, w in zip((a, b), graphs, want):
            for m in s.out():
                m.assign(-3.0)
            c.step()
            g.launch()
            c.step()
            assert all(np.array_equal(p, q) for p, q in zip(bits(s.out()), w)), i
            assert all(np.array_equal(p, q) for p, q in zip(bits(c.out()), want[2])), i
